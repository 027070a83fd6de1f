// Products with one 4-bit or 16-bit weight and the gated feed-forward projections: what runs around linear_kernel, and
// the C-ABI.
//
//   q4_linear   out = dt(x W^T),  dx = dt(dy W),        W = dt(fp16(fp16(q s) + z)) (codec.hip)
//   gated       (G, U) = x W^T,   act = dt(silu(G) U);  kept: dt(G), dt(U), or Q(G), Q(U) in blocks of 128 (fp8.hip)
//               dG = dt(dact U s (1 + G (1 - s))), dU = dt(dact G s), s = sigmoid(G), of the kept values
//               dx = dt([dG, dU] W),   dW = dt([dG, dU]^T x)
//
// The products are linear_kernel's C = A W^T.  A grad-input's weight and both of a weight gradient's operands have the
// contraction's index first: 16-bit ones of whole blocks of 64 are read turned (linear_turned.hip), others from transposed copies
// that the kernels here make in the workspace.
#include "fp8.h"
#include "linear.h"

namespace usaf {
namespace {

constexpr int64_t LIN_MAX = (int64_t)1 << 22;  // columns: 256 rows of 16-bit values stay within 32-bit offsets

int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// ---- copies of operands ----------------------------------------------------------

// 4-bit rows [rows, K] -> 16-bit rows: 8 codes a thread.  28,672 x 4,096: 58 us, 5.1 TB/s, a copy's rate.
template <int DT>
__global__ __launch_bounds__(256) void q4_rows_kernel(const uint32_t* __restrict__ q, const uint32_t* __restrict__ sz,
                                                      int64_t rows, int row_words, u32x4* __restrict__ out) {
  const int64_t stride = (int64_t)gridDim.x * 256, first = (int64_t)blockIdx.x * 256 + threadIdx.x;
  // (a division for each word would take as long as the word)
  const int64_t down = stride / row_words;
  const int right = (int)(stride - down * row_words);
  int64_t n = first / row_words;
  int c = (int)(first - n * row_words);
  for (int64_t i = first; n < rows; i += stride) {
    const uint32_t p = sz[(c >> 4) * rows + n];  // 16 words a group
    const f16 s = __builtin_bit_cast(f16, (uint16_t)p), z = __builtin_bit_cast(f16, (uint16_t)(p >> 16));
    out[i] = dq8<DT>(q[i], f16x2{s, s}, f16x2{z, z});
    n += down;
    c += right;
    if (c >= row_words) {
      c -= row_words;
      ++n;
    }
  }
}

// [S, C] (16-bit, row stride ld; or 4-bit codes, C = K) -> [C, ldo], zeros for s in [S, ldo); ldo % 64 == 0.  A block
// has 64 x 64 values; blocks from `first` on are the second matrix's (16-bit): one launch for both.  28,672 x 4,096 codes: 64 to
// 69 us, 4.3 to 4.6 TB/s; 16,384 x 2,048 and 2,048 x 2,048 16-bit values: 31 to 35, 4.3 to 4.9.
struct Transpose {
  const void* in;
  int64_t S, C, ld;
  uint16_t* out;
  int64_t ldo;
  int wide;  // blocks along S
  bool vec;
};
template <int DT, bool Q4>
__global__ __launch_bounds__(256) void transpose_kernel(const Transpose a, const uint32_t* __restrict__ sz, int64_t first,
                                                        const Transpose b) {
  __shared__ __align__(16) uint32_t tile[TT_DWORDS];
  const bool second = blockIdx.x >= first;  // block-uniform
  const Transpose& t = second ? b : a;
  const int64_t at = blockIdx.x - (second ? first : 0), tall = at / t.wide;
  const int64_t s0 = (at - tall * t.wide) * 64, c0 = tall * 64;
  const int sp = threadIdx.x >> 3, cg = threadIdx.x & 7;
  auto row = [&](int64_t s) -> uint4 {
    const int64_t c = c0 + 8 * cg;
    if (s >= t.S || c >= t.C) return uint4{0, 0, 0, 0};
    if constexpr (Q4) {
      if (!second) {
        const uint32_t w = reinterpret_cast<const uint32_t*>(t.in)[(s * t.C + c) >> 3], p = sz[(c >> 7) * t.S + s];
        const f16 sc = __builtin_bit_cast(f16, (uint16_t)p), z = __builtin_bit_cast(f16, (uint16_t)(p >> 16));
        const u32x4 v = dq8<DT>(w, f16x2{sc, sc}, f16x2{z, z});
        return uint4{v.x, v.y, v.z, v.w};
      }
    }
    const uint16_t* const p = reinterpret_cast<const uint16_t*>(t.in) + s * t.ld + c;
    if (t.vec) return *reinterpret_cast<const uint4*>(p);  // C % 8 == 0
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      w[j] = (c + 2 * j < t.C ? (uint32_t)p[2 * j] : 0u) | (c + 2 * j + 1 < t.C ? (uint32_t)p[2 * j + 1] << 16 : 0u);
    return uint4{w[0], w[1], w[2], w[3]};
  };
  tt_write(tile, sp, cg, row(s0 + 2 * sp), row(s0 + 2 * sp + 1));
  __syncthreads();
#pragma unroll
  for (int it = 0; it < 2; ++it) {
    const int v = threadIdx.x + 256 * it, cl = v >> 3, sg = v & 7;
    if (c0 + cl < t.C) *reinterpret_cast<uint4*>(t.out + (c0 + cl) * t.ldo + s0 + 8 * sg) = tt_read(tile, cl, sg);
  }
}

// [rows, C] -> [rows, ldo] with zeros behind column C; ldo % 8 == 0.  Two matrices of as many columns, one behind the other.
__global__ __launch_bounds__(256) void pad_kernel(const uint16_t* __restrict__ a, int64_t rows_a, int64_t ld_a,
                                                  uint16_t* __restrict__ out_a, const uint16_t* __restrict__ b, int64_t rows_b,
                                                  int64_t ld_b, uint16_t* __restrict__ out_b, int64_t C, int64_t ldo) {
  const int64_t chunks = ldo / 8, n = (rows_a + rows_b) * chunks, stride = (int64_t)gridDim.x * 256;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += stride) {
    const int64_t row = i / chunks, c = 8 * (i - row * chunks);
    const bool second = row >= rows_a;
    const int64_t r = second ? row - rows_a : row;
    const uint16_t* const p = (second ? b + r * ld_b : a + r * ld_a) + c;
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      w[j] = (c + 2 * j < C ? (uint32_t)p[2 * j] : 0u) | (c + 2 * j + 1 < C ? (uint32_t)p[2 * j + 1] << 16 : 0u);
    *reinterpret_cast<uint4*>((second ? out_b : out_a) + r * ldo + c) = uint4{w[0], w[1], w[2], w[3]};
  }
}

// ---- the gated activation's backward ---------------------------------------------

struct GatedBwd {
  const uint16_t* dact;   // [M, I]
  const void* kept;
  const uint8_t* kept_s;
  int64_t M, I, hs;
  bool vec;               // I % 8 == 0 and dact 16-byte aligned
  uint16_t* dgu;          // [M, ldd] = [dG, dU, zeros]
  int64_t ldd;
};

// 8 columns from c on of row m: dG and dU, to dgu too.  Memory bounds it: 4,096 x 14,336 of 8-bit blocks in 77 us (6.1 TB/s),
// 2,048 x 8,192 of 16-bit values with the transpose in 44 (5.3 TB/s).
template <int DT, bool EIGHT>
__device__ __forceinline__ void gated_bwd8(const GatedBwd& g, int64_t m, int64_t c, uint4& dg4, uint4& du4) {
  const int64_t left = g.I - c;
  float da[8], gate[8], up[8], dg[8], du[8];
  load8<DT>(g.dact + m * g.I + c, g.vec, left > 8 ? 8 : (int)left, da);
  if constexpr (EIGHT) {
    const uint8_t* const p = reinterpret_cast<const uint8_t*>(g.kept) + 2 * m * g.hs + c;
    const int64_t nb = g.hs / 128, at = 2 * m * nb + (c >> 7);
    const float sg = __uint_as_float((uint32_t)g.kept_s[at] << 23), su = __uint_as_float((uint32_t)g.kept_s[at + nb] << 23);
    const uint2 g8 = *reinterpret_cast<const uint2*>(p), u8 = *reinterpret_cast<const uint2*>(p + g.hs);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int wg = (int)(j < 2 ? g8.x : g8.y), wu = (int)(j < 2 ? u8.x : u8.y);
      const f32x2 a = j & 1 ? __builtin_amdgcn_cvt_pk_f32_fp8(wg, true) : __builtin_amdgcn_cvt_pk_f32_fp8(wg, false);
      const f32x2 b = j & 1 ? __builtin_amdgcn_cvt_pk_f32_fp8(wu, true) : __builtin_amdgcn_cvt_pk_f32_fp8(wu, false);
      gate[2 * j] = a.x * sg;
      gate[2 * j + 1] = a.y * sg;
      up[2 * j] = b.x * su;
      up[2 * j + 1] = b.y * su;
    }
  } else {
    const uint16_t* const p = reinterpret_cast<const uint16_t*>(g.kept) + 2 * m * g.hs + c;
    unpack8<DT>(*reinterpret_cast<const uint4*>(p), gate);
    unpack8<DT>(*reinterpret_cast<const uint4*>(p + g.hs), up);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * gate[j]));
    dg[j] = da[j] * up[j] * s * (1.0f + gate[j] * (1.0f - s));
    du[j] = da[j] * gate[j] * s;
  }
  dg4 = uint4{pack2<DT>(dg[0], dg[1]), pack2<DT>(dg[2], dg[3]), pack2<DT>(dg[4], dg[5]), pack2<DT>(dg[6], dg[7])};
  du4 = uint4{pack2<DT>(du[0], du[1]), pack2<DT>(du[2], du[3]), pack2<DT>(du[4], du[5]), pack2<DT>(du[6], du[7])};
  uint16_t* const to = g.dgu + m * g.ldd + c;
  if (g.vec) {
    *reinterpret_cast<uint4*>(to) = dg4;
    *reinterpret_cast<uint4*>(to + g.I) = du4;
  } else {
    const uint32_t wg[4] = {dg4.x, dg4.y, dg4.z, dg4.w}, wu[4] = {du4.x, du4.y, du4.z, du4.w};
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < left) {
        to[j] = (uint16_t)(wg[j >> 1] >> (16 * (j & 1)));
        to[g.I + j] = (uint16_t)(wu[j >> 1] >> (16 * (j & 1)));
      }
  }
  if (left <= 8)
    for (int64_t k = 2 * g.I; k < g.ldd; ++k) g.dgu[m * g.ldd + k] = 0;
}

template <int DT, bool EIGHT>
__global__ __launch_bounds__(256) void gated_bwd_kernel(const GatedBwd g) {
  const int64_t chunks = (g.I + 7) / 8, n = g.M * chunks, stride = (int64_t)gridDim.x * 256;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += stride) {
    const int64_t m = i / chunks;
    uint4 dg, du;
    gated_bwd8<DT, EIGHT>(g, m, 8 * (i - m * chunks), dg, du);
  }
}

// The same with dgu's transpose [2 I, mp] beside it (zeros for m in [M, mp), mp % 64 == 0), which the weight gradient
// reads: 64 tokens x 64 columns a block.
template <int DT, bool EIGHT>
__global__ __launch_bounds__(256) void gated_bwd_t_kernel(const GatedBwd g, uint16_t* __restrict__ dgut, int64_t mp, int wide) {
  __shared__ __align__(16) uint32_t tiles[2][TT_DWORDS];
  const int64_t tall = blockIdx.x / wide, m0 = (blockIdx.x - tall * wide) * 64, c0 = tall * 64;
  const int sp = threadIdx.x >> 3, cg = threadIdx.x & 7;
  uint4 dg[2], du[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int64_t m = m0 + 2 * sp + u, c = c0 + 8 * cg;
    dg[u] = du[u] = uint4{0, 0, 0, 0};
    if (m < g.M && c < g.I) gated_bwd8<DT, EIGHT>(g, m, c, dg[u], du[u]);
  }
  tt_write(tiles[0], sp, cg, dg[0], dg[1]);
  tt_write(tiles[1], sp, cg, du[0], du[1]);
  __syncthreads();
#pragma unroll
  for (int it = 0; it < 4; ++it) {
    const int v = threadIdx.x + 256 * (it & 1), cl = v >> 3, sg = v & 7;
    if (c0 + cl < g.I)
      *reinterpret_cast<uint4*>(dgut + ((it >> 1) * g.I + c0 + cl) * mp + m0 + 8 * sg) = tt_read(tiles[it >> 1], cl, sg);
  }
}

// out[m, n] = dt( sum over parts of part[p, m, n] ), in order: 4 columns a thread.  2 x 2,048 x 2,048: 9 us, 4.7 TB/s.
template <int DT>
__global__ __launch_bounds__(256) void join_kernel(const float* __restrict__ part, int parts, int64_t M, int64_t N, int64_t ldp,
                                                   bool vec, uint16_t* __restrict__ out, int64_t ldo) {
  const int64_t chunks = ldp / 4, n = M * chunks, stride = (int64_t)gridDim.x * 256;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += stride) {
    const int64_t m = i / chunks, c = 4 * (i - m * chunks);
    f32x4 v = *reinterpret_cast<const f32x4*>(part + m * ldp + c);
#pragma unroll 4
    for (int p = 1; p < parts; ++p) v += *reinterpret_cast<const f32x4*>(part + (p * M + m) * ldp + c);
    uint16_t* const to = out + m * ldo + c;
    const uint2 w = {pack2<DT>(v.x, v.y), pack2<DT>(v.z, v.w)};
    if (vec) {  // N % 4 == 0
      *reinterpret_cast<uint2*>(to) = w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + j < N) to[j] = (uint16_t)((j < 2 ? w.x : w.y) >> (16 * (j & 1)));
    }
  }
}

unsigned blocks_of(int64_t items, int per) {
  const int64_t b = (items + 256 * per - 1) / (256 * per);
  return (unsigned)(b < 1 ? 1 : b > 65536 ? 65536 : b);
}

int q4_rows(const uint8_t* q, const uint32_t* sz, int64_t rows, int64_t K, int dt, void* out, hipStream_t st) {
  const int64_t words = rows * K / 8;
  if (dt == USAF_BF16)
    q4_rows_kernel<USAF_BF16><<<blocks_of(words, 4), 256, 0, st>>>((const uint32_t*)q, sz, rows, (int)(K / 8), (u32x4*)out);
  else
    q4_rows_kernel<USAF_F16><<<blocks_of(words, 4), 256, 0, st>>>((const uint32_t*)q, sz, rows, (int)(K / 8), (u32x4*)out);
  return check_launch("linear: weight rows");
}

Transpose transpose_of(const void* in, int64_t S, int64_t C, int64_t ld, void* out, int64_t ldo) {
  return {in, S, C, ld, reinterpret_cast<uint16_t*>(out), ldo, (int)(ldo / 64), C % 8 == 0 && ld % 8 == 0 && (uintptr_t)in % 16 == 0};
}
int64_t blocks_of(const Transpose& t) { return t.in ? t.wide * ((t.C + 63) / 64) : 0; }

// a and b, each where its `in` is not null; sz: a is 4-bit codes.
int transpose(const Transpose& a, const uint32_t* sz, const Transpose& b, int dt, hipStream_t st) {
  const int64_t first = blocks_of(a), all = first + blocks_of(b);
  if (all == 0) return USAF_OK;
  if (all > 0x7FFFFFFF) return set_error(USAF_ERR_UNSUPPORTED, "linear: too large a transpose");
  if (!sz) transpose_kernel<USAF_BF16, false><<<(unsigned)all, 256, 0, st>>>(a, sz, first, b);
  else if (dt == USAF_BF16) transpose_kernel<USAF_BF16, true><<<(unsigned)all, 256, 0, st>>>(a, sz, first, b);
  else transpose_kernel<USAF_F16, true><<<(unsigned)all, 256, 0, st>>>(a, sz, first, b);
  return check_launch("linear: transpose");
}

int pad(const void* a, int64_t rows_a, int64_t ld_a, void* out_a, const void* b, int64_t rows_b, int64_t ld_b, void* out_b,
        int64_t C, int64_t ldo, hipStream_t st) {
  pad_kernel<<<blocks_of((rows_a + rows_b) * (ldo / 8), 1), 256, 0, st>>>(
      (const uint16_t*)a, rows_a, ld_a, (uint16_t*)out_a, (const uint16_t*)b, rows_b, ld_b, (uint16_t*)out_b, C, ldo);
  return check_launch("linear: pad");
}

template <int DT, bool EIGHT>
int gated_bwd(const GatedBwd& g, void* dgut, int64_t mp, hipStream_t st) {
  if (dgut) {
    const int64_t wide = mp / 64, blocks = wide * ((g.I + 63) / 64);
    if (blocks > 0x7FFFFFFF) return set_error(USAF_ERR_UNSUPPORTED, "gated_bwd: too large");
    gated_bwd_t_kernel<DT, EIGHT><<<(unsigned)blocks, 256, 0, st>>>(g, reinterpret_cast<uint16_t*>(dgut), mp, (int)wide);
  } else {
    gated_bwd_kernel<DT, EIGHT><<<blocks_of(g.M * ((g.I + 7) / 8), 1), 256, 0, st>>>(g);
  }
  return check_launch("gated_bwd");
}

// C = A W^T of 16-bit operands, contraction K % 64 == 0.
LinArgs product(const void* a, int64_t lda, int64_t M, const void* w, int64_t ldw, int64_t N, int64_t K, void* out, int64_t ldo) {
  LinArgs g{};
  g.A = reinterpret_cast<const uint8_t*>(a);
  g.lda = 2 * lda;
  g.M = M;
  g.K = K;
  g.W = reinterpret_cast<const uint8_t*>(w);
  g.ldw = 2 * ldw;
  g.N = N;
  g.out = reinterpret_cast<uint16_t*>(out);
  g.ldo = ldo;
  return g;
}

// A forward product's sizes, as the plans read them.
LinArgs forward_sizes(int64_t M, int64_t N, int64_t K, bool eight_bit) {
  LinArgs g = product(nullptr, K, M, nullptr, K, N, K, nullptr, 0);
  static uint8_t kept;  // (not read: that there is one decides which tiles may be taken)
  if (eight_bit) g.kept = g.kept_s = &kept;
  return g;
}

// Whether a 4-bit weight of `rows` rows is multiplied as codes; else its 16-bit values are written once, to the workspace, and
// multiplied: 2.5 bytes a weight at about 4 TB/s, and a launch.  Measured (us, as codes / written first, bf16): 128, 512, 1,024,
// 2,048 rows of 4,096 to 4,096 18 / 28, 34 / 39, 46 / 49, 84 / 75; 256, 512, 1,024 of 4,096 to 14,336 44 / 66, 78 / 88,
// 151 / 127; gated, 512 and 1,000 of 2,048 to 5,632 23.7 / 28.3 and 39.2 / 40.7.
bool as_codes(int64_t M, int64_t rows, int64_t K, bool gated, bool eight_bit = false) {
  const LinArgs g = forward_sizes(M, gated ? rows / 2 : rows, K, eight_bit);
  return plan_linear_q4(g, gated).us <= plan_linear_dense(g, gated).us + (double)rows * (double)K * 2.5 / 4e6 + 3;
}

// Pieces of a workspace, each a whole number of 256 bytes.
struct Ws {
  uint8_t* at;
  int64_t used = 0;
  explicit Ws(void* p) : at(reinterpret_cast<uint8_t*>(p)) {}
  void* take(int64_t bytes) {
    void* const p = at ? at + used : nullptr;
    used += round_up(bytes, 256);
    return p;
  }
};

// A product's place for the sums of its parts.  q4: of codes.
struct Parts {
  LinPlan plan;
  void* at;
  int64_t ldp;
  Parts() = default;
  Parts(Ws& ws, int64_t M, int64_t N, int64_t K, bool q4)
      : Parts(ws, M, N, q4 ? plan_linear_q4(sizes(M, N, K), false) : plan_linear_dense(sizes(M, N, K), false)) {}
  Parts(Ws& ws, int64_t M, int64_t N, const LinPlan& of) : plan(of) {
    ldp = round_up(N, 4);
    at = plan.parts > 1 ? ws.take(4 * plan.parts * M * ldp) : nullptr;
  }
  static LinArgs sizes(int64_t M, int64_t N, int64_t K) { return product(nullptr, K, M, nullptr, K, N, K, nullptr, N); }
};

int run(LinArgs g, const Parts& p, int dt, hipStream_t st) {
  g.parts = p.plan.parts;
  g.part = reinterpret_cast<float*>(p.at);
  g.ldp = p.ldp;
  if (int rc = p.plan.launch(g, dt, false, st)) return rc;
  if (g.parts == 1) return clear_error();
  const int64_t items = g.M * (g.ldp / 4);
  const bool vec = g.N % 4 == 0 && g.ldo % 4 == 0 && (uintptr_t)g.out % 8 == 0;
  if (dt == USAF_BF16)
    join_kernel<USAF_BF16><<<blocks_of(items, 1), 256, 0, st>>>(g.part, g.parts, g.M, g.N, g.ldp, vec, g.out, g.ldo);
  else
    join_kernel<USAF_F16><<<blocks_of(items, 1), 256, 0, st>>>(g.part, g.parts, g.M, g.N, g.ldp, vec, g.out, g.ldo);
  return check_launch("linear: sums of the parts");
}

bool sizes_ok(int64_t M, int64_t N, int64_t K) {
  return M >= 0 && M <= 0x7FFFFFFF && N >= 1 && N <= LIN_MAX && K >= 1 && K <= LIN_MAX;
}
bool half_type(int32_t dt) { return dt == USAF_BF16 || dt == USAF_F16; }

struct Q4LinearWs {
  void *w = nullptr, *dy = nullptr;
  Parts parts;
  bool codes;
  int64_t bytes, np;
  Q4LinearWs(void* ws, int64_t M, int64_t N, int64_t K, bool backward) {
    Ws at(ws);
    np = round_up(N, 64);
    codes = !backward && as_codes(M, N, K, false);
    if (backward) {
      w = at.take(2 * K * np);
      if (np != N) dy = at.take(2 * M * np);
      parts = Parts(at, M, K, np, false);
    } else if (!q4_small_ok(M, N, K)) {
      if (!codes) w = at.take(2 * N * K);
      parts = Parts(at, M, N, K, codes);
    }
    bytes = at.used;
  }
};

struct GatedWs {
  void *w = nullptr, *x = nullptr;                                  // forward: 16-bit or padded weight, padded x
  void *dgu = nullptr, *wt = nullptr, *dgut = nullptr, *xt = nullptr;  // backward
  Parts dx_parts, dw_parts;
  bool codes = false, dx_turned = false, dw_turned = false;
  int64_t bytes, kp, ldd, mp;
  // what: 0 forward, 4 forward that keeps 8-bit blocks, else 1 for dx + 2 for dw
  GatedWs(void* ws, int64_t M, int64_t I, int64_t K, bool four_bit, int what) {
    Ws at(ws);
    kp = round_up(K, 64);
    ldd = round_up(2 * I, 64);
    mp = round_up(M, 64);
    if ((what & 3) == 0) {
      codes = four_bit && (q4_small_ok(M, I, K) || as_codes(M, 2 * I, K, true, what == 4));
      if (four_bit ? !codes : kp != K) w = at.take(2 * 2 * I * kp);
      if (kp != K) x = at.take(2 * M * kp);
    } else {
      // Operands are read turned where the rows are whole blocks of 64 and chunks of 8 and that is shorter than the product of
      // copies and the copies, 4 bytes a value at about 4 TB/s (dgu's is written with it) and a launch.  Measured (us, dx and dW,
      // turned / copies, tokens x I x K, bf16): 2,048 x 8,192 x 2,048 280 / 324, 512 x 2,816 x 2,048 50 / 59, 64 x 8,192 x 2,048 46 / 66,
      // 4,096 x 14,336 x 4,096 1,572 / 1,732; dW alone, few tiles of a long contraction, 65,536 x 64 x 64 45 / 35; 8,192 x 256 x 256
      // 24.7 / 22.8, on the wrong side
      dgu = at.take(2 * M * ldd);
      if (what & 1) {
        const LinArgs g = Parts::sizes(M, K, ldd);
        const LinPlan turned = plan_linear_turned(g, false);
        dx_turned = !four_bit && ldd == 2 * I && K % 8 == 0 &&
                    turned.us <= plan_linear_dense(g, false).us + (double)K * (double)ldd * 4 / 4e6 + 3;
        if (!dx_turned) wt = at.take(2 * K * ldd);
        dx_parts = dx_turned ? Parts(at, M, K, turned) : Parts(at, M, K, ldd, false);
      }
      if (what & 2) {
        const LinArgs g = Parts::sizes(2 * I, K, mp);
        const LinPlan turned = plan_linear_turned(g, true);
        dw_turned = mp == M && I % 4 == 0 && K % 8 == 0 &&
                    turned.us <= plan_linear_dense(g, false).us + (double)M * (double)(2 * K + 2 * I) * 2 / 4e6 +
                                     ((what & 1) && !dx_turned ? 0 : 3);
        if (!dw_turned) {
          dgut = at.take(2 * 2 * I * mp);
          xt = at.take(2 * K * mp);
        }
        dw_parts = dw_turned ? Parts(at, 2 * I, K, turned) : Parts(at, 2 * I, K, mp, false);
      }
    }
    bytes = at.used;
  }
};

int check_ws(const char* what, const void* ws, int64_t have, int64_t need) {
  if (need && (!ws || (uintptr_t)ws % 16 || have < need))
    return set_error(USAF_ERR_INVALID, "%s: a workspace of %lld bytes, 16-byte aligned, got %lld", what, (long long)need,
                     (long long)have);
  return USAF_OK;
}

}  // namespace

void prepare_linear_kernels() {
  prepare_linear_dense();
  prepare_linear_q4();
  prepare_linear_turned();
  prepare_q4_small();
}

}  // namespace usaf

using namespace usaf;

extern "C" int64_t usaf_hip_q4_linear_ws_bytes(int64_t M, int64_t N, int64_t K, int32_t backward) {
  return sizes_ok(M, N, K) ? Q4LinearWs(nullptr, M, N, K, backward != 0).bytes : -1;
}

static int q4_args(const char* what, const void* a, int32_t dtype, int64_t M, int64_t N, int64_t K, int64_t ld, int64_t cols,
                   const uint8_t* q, const uint32_t* sz, const void* out) {
  if (!sizes_ok(M, N, K) || K % 128)
    return set_error(USAF_ERR_INVALID, "%s: need M >= 0, 1 <= N, K <= %lld and K %% 128 == 0, got M=%lld N=%lld K=%lld", what,
                     (long long)LIN_MAX, (long long)M, (long long)N, (long long)K);
  if (!half_type(dtype)) return set_error(USAF_ERR_INVALID, "%s: dtype must be fp16 or bf16", what);
  if (M == 0) return USAF_OK;
  if (!a || !q || !sz || !out) return set_error(USAF_ERR_INVALID, "%s: null pointer", what);
  if (ld < cols || ld > LIN_MAX) return set_error(USAF_ERR_INVALID, "%s: rows of %lld values, %lld apart", what, (long long)cols, (long long)ld);
  if ((uintptr_t)q % 16 || (uintptr_t)sz % 4 || ((uintptr_t)out | (uintptr_t)a) % 2)
    return set_error(USAF_ERR_INVALID, "%s: codes must be 16-byte, scales 4-byte, rows and output 2-byte aligned", what);
  return USAF_OK;
}

extern "C" int usaf_hip_q4_linear(const void* x, int32_t dtype, int64_t M, int64_t K, int64_t ld, const uint8_t* q,
                                  const uint32_t* sz, int64_t N, void* out, void* ws, int64_t ws_bytes, void* stream) {
  if (int rc = q4_args("q4_linear", x, dtype, M, N, K, ld, K, q, sz, out)) return rc;
  if (M == 0) return clear_error();
  if ((uintptr_t)x % 16 || ld % 8) return set_error(USAF_ERR_INVALID, "q4_linear: rows must be 16-byte aligned");
  const Q4LinearWs w(ws, M, N, K, false);
  if (int rc = check_ws("q4_linear", ws, ws_bytes, w.bytes)) return rc;
  hipStream_t st = as_stream(stream);
  if (w.codes || q4_small_ok(M, N, K)) {
    LinArgs g = product(x, ld, M, q, 0, N, K, out, N);
    g.ldw = K / 2;
    g.sz = sz;
    if (q4_small_ok(M, N, K)) return q4_small(g, dtype, false, st);
    return run(g, w.parts, dtype, st);
  }
  if (int rc = q4_rows(q, sz, N, K, dtype, w.w, st)) return rc;
  return run(product(x, ld, M, w.w, K, N, K, out, N), w.parts, dtype, st);
}

extern "C" int usaf_hip_q4_linear_bwd(const void* dy, int32_t dtype, int64_t M, int64_t N, int64_t ld, const uint8_t* q,
                                      const uint32_t* sz, int64_t K, void* dx, void* ws, int64_t ws_bytes, void* stream) {
  if (int rc = q4_args("q4_linear_bwd", dy, dtype, M, N, K, ld, N, q, sz, dx)) return rc;
  if (M == 0) return clear_error();
  const Q4LinearWs w(ws, M, N, K, true);
  if (int rc = check_ws("q4_linear_bwd", ws, ws_bytes, w.bytes)) return rc;
  if (!w.dy && ((uintptr_t)dy % 16 || ld % 8)) return set_error(USAF_ERR_INVALID, "q4_linear_bwd: rows must be 16-byte aligned");
  hipStream_t st = as_stream(stream);
  if (int rc = transpose(transpose_of(q, N, K, K, w.w, w.np), sz, Transpose{}, dtype, st)) return rc;
  if (w.dy)
    if (int rc = pad(dy, M, ld, w.dy, nullptr, 0, 0, nullptr, N, w.np, st)) return rc;
  return run(product(w.dy ? w.dy : dy, w.dy ? w.np : ld, M, w.w, w.np, K, w.np, dx, K), w.parts, dtype, st);
}

static int gated_args(const char* what, int32_t dtype, int64_t M, int64_t I, int64_t K, const uint8_t* q, const uint32_t* sz,
                      const void* w16) {
  if (!sizes_ok(M, 2 * I, K))
    return set_error(USAF_ERR_INVALID, "%s: need M >= 0 and 1 <= 2 I, K <= %lld, got M=%lld I=%lld K=%lld", what, (long long)LIN_MAX,
                     (long long)M, (long long)I, (long long)K);
  if (!half_type(dtype)) return set_error(USAF_ERR_INVALID, "%s: dtype must be fp16 or bf16", what);
  if (M == 0) return USAF_OK;
  if ((q == nullptr) == (w16 == nullptr) || (q && !sz))
    return set_error(USAF_ERR_INVALID, "%s: a 4-bit weight (codes and scales) or a 16-bit one", what);
  if (((uintptr_t)q | (uintptr_t)w16) % 16 || (uintptr_t)sz % 4)
    return set_error(USAF_ERR_INVALID, "%s: weights must be 16-byte, scales 4-byte aligned", what);
  if (q && K % 128) return set_error(USAF_ERR_INVALID, "%s: a 4-bit weight's K must be a multiple of 128, got %lld", what, (long long)K);
  if (q && (I + 256) * (K / 2) >= (int64_t)1 << 32)
    return set_error(USAF_ERR_UNSUPPORTED, "%s: a gate of 4 GiB of codes", what);
  return USAF_OK;
}

extern "C" int64_t usaf_hip_gated_ws_bytes(int64_t M, int64_t I, int64_t K, int32_t four_bit, int32_t what) {
  return sizes_ok(M, 2 * I, K) && what >= 0 && what <= 4 ? GatedWs(nullptr, M, I, K, four_bit != 0, what).bytes : -1;
}

// {kind, tile's rows, tile's weight rows, parts of the contraction}
static int tell(int32_t* to, int kind, const LinPlan& p) {
  const int32_t v[4] = {kind, p.rows, p.w_rows, p.parts};
  for (int i = 0; i < 4; ++i) to[i] = v[i];
  return clear_error();
}
static const LinPlan FEW_ROWS{nullptr, 1, 0, 16, 16};

extern "C" int usaf_hip_q4_linear_plan(int64_t M, int64_t N, int64_t K, int32_t backward, int32_t* plan) {
  if (!sizes_ok(M, N, K) || M == 0 || !plan) return set_error(USAF_ERR_INVALID, "q4_linear_plan: sizes or a null pointer");
  if (!backward && q4_small_ok(M, N, K)) return tell(plan, USAF_PLAN_FEW_ROWS, FEW_ROWS);
  const Q4LinearWs w(nullptr, M, N, K, backward != 0);
  return tell(plan, w.codes ? USAF_PLAN_CODES : USAF_PLAN_ROWS, w.parts.plan);
}

extern "C" int usaf_hip_gated_plan(int64_t M, int64_t I, int64_t K, int32_t four_bit, int32_t what, int32_t weight_grad,
                                   int32_t* plan) {
  const bool forward = what == 0 || what == 4;
  if (!sizes_ok(M, 2 * I, K) || M == 0 || !plan || what < 0 || what > 4 || (!forward && !(what & (weight_grad ? 2 : 1))))
    return set_error(USAF_ERR_INVALID, "gated_plan: sizes, what or a null pointer");
  const GatedWs w(nullptr, M, I, K, four_bit != 0, what);
  if (!forward)
    return weight_grad ? tell(plan, w.dw_turned ? USAF_PLAN_BOTH_TURNED : USAF_PLAN_ROWS, w.dw_parts.plan)
                       : tell(plan, w.dx_turned ? USAF_PLAN_W_TURNED : USAF_PLAN_ROWS, w.dx_parts.plan);
  if (w.codes && what == 0 && q4_small_ok(M, I, K)) return tell(plan, USAF_PLAN_FEW_ROWS, FEW_ROWS);
  const LinArgs g = forward_sizes(M, I, w.kp, what == 4);
  return w.codes ? tell(plan, USAF_PLAN_CODES, plan_linear_q4(g, true)) : tell(plan, USAF_PLAN_ROWS, plan_linear_dense(g, true));
}

extern "C" int usaf_hip_gated_fwd(const void* x, int32_t dtype, int64_t M, int64_t K, int64_t ld, const uint8_t* q,
                                  const uint32_t* sz, const void* w16, int64_t I, void* act, void* kept, uint8_t* kept_scales,
                                  void* ws, int64_t ws_bytes, void* stream) {
  if (int rc = gated_args("gated_fwd", dtype, M, I, K, q, sz, w16)) return rc;
  if (M == 0) return clear_error();
  if (!x || !act || (kept_scales && !kept)) return set_error(USAF_ERR_INVALID, "gated_fwd: null pointer");
  if (ld < K || ld > LIN_MAX) return set_error(USAF_ERR_INVALID, "gated_fwd: rows of %lld values, %lld apart", (long long)K, (long long)ld);
  const GatedWs w(ws, M, I, K, q != nullptr, kept_scales ? 4 : 0);
  if ((uintptr_t)kept % 16 || (uintptr_t)act % 2 || (!w.x && ((uintptr_t)x % 16 || ld % 8)) || (uintptr_t)x % 2)
    return set_error(USAF_ERR_INVALID, "gated_fwd: rows and what is kept must be 16-byte aligned");
  if (int rc = check_ws("gated_fwd", ws, ws_bytes, w.bytes)) return rc;
  hipStream_t st = as_stream(stream);
  if (w.x)  // (then the weight is a 16-bit one, padded as well)
    if (int rc = pad(x, M, ld, w.x, w16, 2 * I, K, w.w, K, w.kp, st)) return rc;
  LinArgs g = product(w.x ? w.x : x, w.x ? w.kp : ld, M, w.w ? w.w : w16, w.kp, I, w.kp, act, I);
  g.kept = kept;
  g.kept_s = kept_scales;
  g.hs = round_up(I, kept_scales ? 128 : 8);
  if (q && !w.w) {
    g.W = q;
    g.ldw = K / 2;
    g.sz = sz;
    if (!kept && q4_small_ok(M, I, K)) return q4_small(g, dtype, true, st);
    return plan_linear_q4(g, true).launch(g, dtype, true, st);
  }
  if (q)
    if (int rc = q4_rows(q, sz, 2 * I, K, dtype, w.w, st)) return rc;
  return plan_linear_dense(g, true).launch(g, dtype, true, st);
}

extern "C" int usaf_hip_gated_bwd(const void* dact, int32_t dtype, int64_t M, int64_t I, int64_t K, const void* kept,
                                  const uint8_t* kept_scales, const uint8_t* q, const uint32_t* sz, const void* w16,
                                  const void* x, int64_t ldx, void* dx, void* dw, void* ws, int64_t ws_bytes, void* stream) {
  if (int rc = gated_args("gated_bwd", dtype, M, I, K, q, sz, w16)) return rc;
  if (M == 0) return clear_error();
  if (!dact || !kept || (!dx && !dw) || (dw && !x)) return set_error(USAF_ERR_INVALID, "gated_bwd: null pointer");
  if (dw && q) return set_error(USAF_ERR_INVALID, "gated_bwd: a 4-bit weight has no gradient");
  // (x read turned has 32-bit offsets within 64 rows)
  if (dw && (ldx < K || ldx > LIN_MAX || M > LIN_MAX))
    return set_error(USAF_ERR_INVALID, "gated_bwd: a weight gradient needs K <= ldx <= %lld and M <= %lld, got ldx=%lld M=%lld",
                     (long long)LIN_MAX, (long long)LIN_MAX, (long long)ldx, (long long)M);
  if ((uintptr_t)kept % 16 || ((uintptr_t)dact | (uintptr_t)x | (uintptr_t)dx | (uintptr_t)dw) % 2)
    return set_error(USAF_ERR_INVALID, "gated_bwd: what is kept must be 16-byte, rows 2-byte aligned");
  const GatedWs w(ws, M, I, K, q != nullptr, (dx ? 1 : 0) | (dw ? 2 : 0));
  if (w.dw_turned && ((uintptr_t)x % 16 || ldx % 8)) return set_error(USAF_ERR_INVALID, "gated_bwd: rows of x must be 16-byte aligned");
  if (int rc = check_ws("gated_bwd", ws, ws_bytes, w.bytes)) return rc;
  hipStream_t st = as_stream(stream);
  GatedBwd g{reinterpret_cast<const uint16_t*>(dact), kept, kept_scales, M, I, round_up(I, kept_scales ? 128 : 8),
             I % 8 == 0 && (uintptr_t)dact % 16 == 0, reinterpret_cast<uint16_t*>(w.dgu), w.ldd};
  const int rc = dtype == USAF_BF16
                     ? (kept_scales ? gated_bwd<USAF_BF16, true>(g, w.dgut, w.mp, st) : gated_bwd<USAF_BF16, false>(g, w.dgut, w.mp, st))
                     : (kept_scales ? gated_bwd<USAF_F16, true>(g, w.dgut, w.mp, st) : gated_bwd<USAF_F16, false>(g, w.dgut, w.mp, st));
  if (rc) return rc;
  const Transpose wt = w.wt ? transpose_of(q ? (const void*)q : w16, 2 * I, K, K, w.wt, w.ldd) : Transpose{};
  const Transpose xt = w.xt ? transpose_of(x, M, K, ldx, w.xt, w.mp) : Transpose{};
  if (int rc2 = transpose(wt, q ? sz : nullptr, xt, dtype, st)) return rc2;
  if (dx)
    if (int rc2 = run(w.dx_turned ? product(w.dgu, w.ldd, M, w16, K, K, w.ldd, dx, K)
                                  : product(w.dgu, w.ldd, M, w.wt, w.ldd, K, w.ldd, dx, K), w.dx_parts, dtype, st)) return rc2;
  if (dw)
    return run(w.dw_turned ? product(w.dgu, w.ldd, 2 * I, x, ldx, K, w.mp, dw, K)
                           : product(w.dgut, w.mp, 2 * I, w.xt, w.mp, K, w.mp, dw, K), w.dw_parts, dtype, st);
  return clear_error();
}

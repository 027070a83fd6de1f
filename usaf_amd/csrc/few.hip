// A whole MoE layer for 1 to 32 tokens, on 4-bit or 8-bit experts:
//
//   l = x Wr^T, the k largest l (ties: the lowest expert), w = softmax(l) there (renormalised or not)
//   a_e = dt(silu(g) u),  (g, u) = Wgu_e x;   out = dt(sum_e w_e Wd_e a_e)
//
// Four launches (three for one or two tokens), nothing read back to the host, no slot lists:
//
//   few_logits   a block an expert of the router and up to four tokens
//   few_route    a wave a token: the k largest, their weights, a bit of the token in their masks (one or two tokens: in
//                few_gate_up)
//   few_gate_up  a block takes (expert in use, 32 columns of a) tiles; its waves split the contraction
//   few_down     a block has 64 columns of out; the waves of a column tile share its (expert,
//                group of 128) pairs evenly and add them up by token; the tile's last block adds the parts in order
//
// An expert's tokens are the rows of a 16-row MFMA operand (more than 16: a second
// round), weights its columns: a lane has one weight row and four tokens, so a row's scale
// and zero are one register each.  A group of 128 is multiplied as codes, D = sum_k x_k
// (c_k + offset) with exact small whole numbers as operands, and
//   y += s D + (z - offset s) sum_k x_k           (4-bit; the sum by an MFMA against ones)
//   y += 2^e D                                    (8-bit)
// which takes 7 vector instructions for 8 codes and 8 for a group of 16 rows, where
// dequantizing each weight takes 32 for 8 codes.  The weight is the real number s q + z: nothing
// rounds it.
#include "fp8.h"

namespace usaf {
namespace {

constexpr int FT = 32;        // tokens at most
constexpr int FR = 16;        // tokens of one operand
constexpr int F_MAX_E = 256;  // experts
constexpr int F_MAX_K = 16;   // experts of a token
enum { FMT_Q4 = 0, FMT_FP8 = 1 };

struct FewArgs {
  const uint16_t* x;        // [T, H]
  const uint16_t* router;   // [E, H]
  int T, E, k, norm;
  int H, I;
  const uint8_t* gu;        // codes [E, 2I, H]
  const void* gu_s;         // 4-bit: fp16 scale | zero << 16, [E, H / 128, 2I]; 8-bit: E8M0 bytes
  const uint8_t* dn;        // codes [E, H, I]
  const void* dn_s;
  uint16_t* out;            // [T, H]
  // workspace
  double* logits;           // [T, E]
  uint32_t* mask;           // [F_MAX_E] tokens of each expert
  float* wt;                // [E, FT] their weights
  uint16_t* xp;             // [T, H] x in the fragments' order (4-bit)
  uint16_t* act;            // [experts in use, T, I] in the fragments' order
  float* part;              // [P, T, H] partial sums
  int32_t* done;            // [H / 64] parts of a column tile that have arrived
  int P;                    // few_down: blocks of a column tile
};

// Order of 8 neighbouring values in a fragment of 4-bit codes: a code word's nibbles
// come apart as (0, 4), (1, 5), (2, 6), (3, 7).
template <int FMT>
__device__ __forceinline__ int frag_pos(int c) {
  if constexpr (FMT == FMT_Q4) return (c & ~7) | ((c & 3) << 1) | ((c >> 2) & 1);
  else return c;
}

// ---- routing ---------------------------------------------------------------------

// A total order of doubles: larger is larger, a NaN below everything.
__device__ __forceinline__ int64_t order_key(double v) {
  if (v != v) return INT64_MIN;
  const int64_t b = __double_as_longlong(v);
  return b < 0 ? -(b & INT64_MAX) : b;  // -0 with 0
}

// logits[t, e], products of 8 in fp32 and their sums in 64 bits: which expert is the
// k-th hangs on differences near fp32's own rounding.  Block: one expert and TB tokens, a quarter
// of a row for each wave, so that rows of 2,048 are one load deep: 3.0 us for one token and 128 experts,
// 4.7 for 24, a launch and one trip to memory (a wave a row took 4.3 and 8.1).
template <int DT, int FMT, int TB>
__global__ __launch_bounds__(256) void few_logits_kernel(const FewArgs g) {
  __shared__ double s_part[4][TB];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int tb = blockIdx.x / g.E, e = blockIdx.x - tb * g.E, t0 = tb * TB;
  const uint16_t* const wr = g.router + (int64_t)e * g.H;
  const uint16_t* xr[TB];
#pragma unroll
  for (int i = 0; i < TB; ++i) xr[i] = g.x + (int64_t)(t0 + i < g.T ? t0 + i : g.T - 1) * g.H;
  double acc[TB];
#pragma unroll
  for (int i = 0; i < TB; ++i) acc[i] = 0;
#pragma unroll 2
  for (int h = 8 * tid; h < g.H; h += 2048) {
    const uint4 w = *reinterpret_cast<const uint4*>(wr + h);
    const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < TB; ++i) {
      const uint4 v = *reinterpret_cast<const uint4*>(xr[i] + h);
      const uint32_t xw[4] = {v.x, v.y, v.z, v.w};
      float s = 0.f;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x2 a = unpack2<DT>(xw[q]), b = unpack2<DT>(ww[q]);
        s = fmaf(a.x, b.x, s);
        s = fmaf(a.y, b.y, s);
      }
      acc[i] += (double)s;
    }
  }
  // what the later launches start from, while the loads are on their way
  const int id = blockIdx.x * 256 + tid, threads = gridDim.x * 256;
  for (int i = id; i < F_MAX_E; i += threads) g.mask[i] = 0;
  for (int i = id; i < g.H / 64; i += threads) g.done[i] = 0;
  if constexpr (FMT == FMT_Q4) {
    for (int i = id; i < g.T * (g.H / 8); i += threads) {
      const uint4 v = *reinterpret_cast<const uint4*>(g.x + 8 * (int64_t)i);
      const uint4 o = {__builtin_amdgcn_perm(v.z, v.x, 0x05040100u), __builtin_amdgcn_perm(v.z, v.x, 0x07060302u),
                       __builtin_amdgcn_perm(v.w, v.y, 0x05040100u), __builtin_amdgcn_perm(v.w, v.y, 0x07060302u)};
      *reinterpret_cast<uint4*>(g.xp + 8 * (int64_t)i) = o;
    }
  }
  // a token's sum in the 64 / TB lanes that keep it: a quarter each of four tokens, half the shuffles at every step
  int at = 0;
  if constexpr (TB == 4) {
    const bool up = lane & 32, odd = lane & 16;
    const double a = (up ? acc[2] : acc[0]) + __shfl_xor(up ? acc[0] : acc[2], 32, 64);
    const double b = (up ? acc[3] : acc[1]) + __shfl_xor(up ? acc[1] : acc[3], 32, 64);
    acc[0] = (odd ? b : a) + __shfl_xor(odd ? a : b, 16, 64);
    at = lane >> 4;
  } else {
    acc[0] += __shfl_xor(acc[0], 32, 64);
    acc[0] += __shfl_xor(acc[0], 16, 64);
  }
#pragma unroll
  for (int d = 8; d > 0; d >>= 1) acc[0] += __shfl_xor(acc[0], d, 64);
  if ((lane & 15) == 0 && (TB == 4 || lane == 0)) s_part[wave][at] = acc[0];
  __syncthreads();
  if (tid < TB && t0 + tid < g.T)
    g.logits[(int64_t)(t0 + tid) * g.E + e] = (s_part[0][tid] + s_part[1][tid]) + (s_part[2][tid] + s_part[3][tid]);
}

// As order_key, and no two alike: the lowest 8 of a double's 52 bits give way to the expert's
// number (logits are not known that well), the lower number first.
__device__ __forceinline__ int64_t expert_key(double v, int e) { return (order_key(v) & ~(int64_t)255) | (255 - e); }

__device__ __forceinline__ float rows16_max(float v) {  // of a wave's lanes, each row of 16 its own already
  const float a = fmaxf(__shfl(v, 0, 64), __shfl(v, 16, 64)), b = fmaxf(__shfl(v, 32, 64), __shfl(v, 48, 64));
  return fmaxf(a, b);
}
template <int N>
__device__ __forceinline__ float add_rot(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 + N, 0xf, 0xf, false));
}
__device__ __forceinline__ float wave_add(float v) {  // the same bits in every lane
  v = add_rot<1>(add_rot<2>(add_rot<4>(add_rot<8>(v))));
  return (__shfl(v, 0, 64) + __shfl(v, 16, 64)) + (__shfl(v, 32, 64) + __shfl(v, 48, 64));
}

template <int N>
__device__ __forceinline__ int max_rot_i(int v) {
  const int o = __builtin_amdgcn_update_dpp(0, v, 0x120 + N, 0xf, 0xf, false);
  return o > v ? o : v;
}
__device__ __forceinline__ int wave_max_i(int v) {  // uniform
  v = max_rot_i<1>(max_rot_i<2>(max_rot_i<4>(max_rot_i<8>(v))));
  const int a = __builtin_amdgcn_readlane(v, 0), b = __builtin_amdgcn_readlane(v, 16);
  const int c = __builtin_amdgcn_readlane(v, 32), d = __builtin_amdgcn_readlane(v, 48);
  const int x = a > b ? a : b, y = c > d ? c : d;
  return x > y ? x : y;
}

// The first k experts of a token, by one wave: up to four experts a lane, the largest key taken k
// times, by its upper half first: 2 us for 8 of 128 (counting how many come before each expert: 3.7).
struct Chosen {
  static constexpr int N = F_MAX_E / 64;
  double l[N];
  int rank[N];  // -1: not chosen
  __device__ __forceinline__ Chosen(const double* row, int E, int k, int lane) {
    int high[N], low[N];  // low: the unsigned order as a signed one
#pragma unroll
    for (int i = 0; i < N; ++i) l[i] = 64 * i + lane < E ? row[64 * i + lane] : -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int64_t key = 64 * i + lane < E ? expert_key(l[i], 64 * i + lane) : INT64_MIN;
      high[i] = (int)(key >> 32);
      low[i] = (int)((uint32_t)key ^ 0x80000000u);
      rank[i] = -1;
    }
    for (int n = 0; n < k; ++n) {
      int m = high[0], at = 0;
#pragma unroll
      for (int i = 1; i < N; ++i) m = high[i] > m ? high[i] : m;
      m = wave_max_i(m);
      bool first[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        first[i] = high[i] == m;
        at += __popcll(__ballot(first[i]));
      }
      if (at > 1) {  // uniform
        int q = INT32_MIN;
#pragma unroll
        for (int i = 0; i < N; ++i) q = first[i] && low[i] > q ? low[i] : q;
        q = wave_max_i(q);
#pragma unroll
        for (int i = 0; i < N; ++i) first[i] = first[i] && low[i] == q;
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {  // taken: below all others from here on
        rank[i] = first[i] ? n : rank[i];
        high[i] = first[i] ? INT32_MIN : high[i];
        low[i] = first[i] ? INT32_MIN : low[i];
      }
    }
  }
  // Their weights to g.wt; s_p: room for k, the wave's own.
  __device__ __forceinline__ void weights(const FewArgs& g, int t, int lane, float* s_p) const {
    float m = -INFINITY, sum = 0.f, p[N];
#pragma unroll
    for (int i = 0; i < N; ++i) m = fmaxf(m, (float)l[i]);
    m = rows16_max(max16(m));
#pragma unroll
    for (int i = 0; i < N; ++i) {
      p[i] = 64 * i + lane < g.E ? expf((float)(l[i] - (double)m)) : 0.f;
      sum += p[i];
      if (rank[i] >= 0) s_p[rank[i]] = p[i];
    }
    sum = wave_add(sum);
    __builtin_amdgcn_wave_barrier();  // one wave's LDS operations complete in order
    float total = sum;
    if (g.norm) {
      total = 0.f;
      for (int i = 0; i < g.k; ++i) total += s_p[i];
      if (sum != sum) total = sum;  // a NaN anywhere in the row
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (rank[i] >= 0) g.wt[(64 * i + lane) * FT + t] = p[i] / total;
  }
};

// Block: one token, one wave: 4.8 us for 24 tokens and 128 experts, a launch, one trip to memory and the choice.
__global__ __launch_bounds__(64) void few_route_kernel(const FewArgs g) {
  __shared__ float s_p[F_MAX_K];
  const int t = blockIdx.x, lane = threadIdx.x;
  const Chosen c(g.logits + (int64_t)t * g.E, g.E, g.k, lane);
  c.weights(g, t, lane, s_p);
#pragma unroll
  for (int i = 0; i < Chosen::N; ++i)
    if (c.rank[i] >= 0) atomicOr(&g.mask[64 * i + lane], 1u << t);  // bits of different blocks: any order gives the same mask
}

// ---- products --------------------------------------------------------------------

// Place of the n-th set bit.
__device__ __forceinline__ int nth_bit(uint32_t m, int n) {
  int at = 0;
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) {
    const int c = __popc((m >> at) & ((1u << w) - 1));
    const bool past = n >= c;
    n -= past ? c : 0;
    at += past ? w : 0;
  }
  return at;
}
__device__ __forceinline__ int nth_bit(uint64_t m, int n) {
  const int low = __popc((uint32_t)m);
  return n < low ? nth_bit((uint32_t)m, n) : 32 + nth_bit((uint32_t)(m >> 32), n - low);
}

// An expert and up to 16 of its tokens: what one pass over its weights multiplies.
struct Item {
  int e, u;         // the expert, its place among those in use
  uint32_t tokens;  // all its tokens
  int b;            // which 16 of them
};

// The experts in use, held by a wave: their bits, those of experts with more than 16
// tokens (which come again behind all others), and the lane's four masks.
struct InUse {
  static constexpr int N = F_MAX_E / 64;
  uint64_t bits[N], more[N];
  uint32_t mask[N];
  int count, items;
  __device__ __forceinline__ void load(const uint32_t* m, int lane) {
#pragma unroll
    for (int i = 0; i < N; ++i) mask[i] = m[64 * i + lane];
    find();
  }
  __device__ __forceinline__ void find() {
    count = items = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      bits[i] = __ballot(mask[i] != 0);
      more[i] = __ballot(__popc(mask[i]) > FR);
      count += __popcll(bits[i]);
      items += __popcll(more[i]);
    }
    items += count;
  }
  // Item i < items; everything uniform.
  __device__ __forceinline__ Item item(int i) const {
    Item t;
    t.b = i >= count;
    int n = t.b ? i - count : i, before = 0;
    t.e = t.u = 0;
    t.tokens = 0;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const uint64_t from = t.b ? more[k] : bits[k];
      const int c = __popcll(from);
      if (n >= 0 && n < c) {
        const int at = __builtin_amdgcn_readfirstlane(nth_bit(from, n));
        t.e = 64 * k + at;
        t.u = before + __popcll(bits[k] & ((1ull << at) - 1));
        t.tokens = (uint32_t)__builtin_amdgcn_readlane((int)mask[k], at);
      }
      n -= c;
      before += __popcll(bits[k]);
    }
    return t;
  }
};

// A wave multiplies in steps: 128 bytes of each of its weight rows, two groups of 4-bit
// codes or one of 8-bit ones, by units of 16 rows.  As soon as the codes of a step have left
// their registers for LDS, those of the next step are loaded there: a wave has a whole step's
// weights in flight behind its arithmetic.
//
// The codes come as they lie in memory, neighbouring lanes at neighbouring 16 bytes, whole
// 128-byte lines, and reach the fragments through LDS.  Loaded straight into fragments
// (lanes 0 to 15 in 16 rows) each lane's 16 bytes are an access of their own to the address
// unit, 48 a load, and steps of half a line ask the memory for 64 bytes at a time: gate_up of
// 24 tokens took 55 us, and 41 with the first of the two mended.
template <int FMT>
constexpr int STEP = FMT == FMT_Q4 ? 2 : 1;  // groups
constexpr int UNIT_LDS = 2048;

template <int FMT>
struct Unit {
  u32x4 c[2];             // codes: lane l has word l % 8 of rows l / 8 and 8 + l / 8
  uint32_t z[STEP<FMT>];  // scale | zero of row l % 16, or the E8M0 byte
};
struct Values {           // tokens, one group: lane (r, q), register j: k = 32 q + 8 j + [0, 8) of token row r
  u32x4 x[4];
};

typedef __amdgpu_buffer_rsrc_t Buffer;
// Loads past `bytes` give zeros and touch no memory: what lanes of unused token rows do.
__device__ __forceinline__ Buffer buffer_of(const void* p, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, bytes, 0x00020000);
}
constexpr uint32_t NO_ROW = 0x80000000u;  // past any buffer here
constexpr int DEVICE_SCOPE = 16;          // sc1 of a buffer instruction

// Where a wave's operands of a step come from: for each unit the first weight row's codes
// and scales, wave-uniform, and the tokens; the lane's place in them as byte offsets.
template <int NU>
struct Source {
  const uint8_t* w[NU];
  const uint8_t* s[NU];
  Buffer x;
  uint32_t x_off;

  // Units of rows row[v] + [0, 16) of expert e's [R, K] matrix.  Scales: 4-bit [E, K / 128, R]
  // words, 8-bit [E, ceil(R / 128), K / 128] bytes.
  template <int FMT>
  __device__ __forceinline__ void weights(const uint8_t* codes, const void* scales, int e, int R, int K,
                                          const int (&row)[NU]) {
    const int ng = K / 128;
    const int64_t rb = FMT == FMT_Q4 ? K / 2 : K;
#pragma unroll
    for (int v = 0; v < NU; ++v) {
      w[v] = codes + ((int64_t)e * R + row[v]) * rb;
      if constexpr (FMT == FMT_Q4) s[v] = reinterpret_cast<const uint8_t*>(scales) + ((int64_t)e * ng * R + row[v]) * 4;
      else s[v] = reinterpret_cast<const uint8_t*>(scales) + ((int64_t)e * ((R + 127) / 128) + row[v] / 128) * ng;
    }
  }
};

// The lane's place in a step of a unit, as byte offsets (R rows of K).
template <int FMT>
struct Place {
  uint32_t whole, last;  // codes; of a row's last group alone (4-bit, an odd number of groups): its words twice
  uint32_t z;
  int64_t rows8;         // bytes of 8 rows
  int ng, R;
  __device__ __forceinline__ Place(int R_, int K, int lane) : ng(K / 128), R(R_) {
    const int rb = FMT == FMT_Q4 ? K / 2 : K;
    whole = (uint32_t)((lane >> 3) * rb + 16 * (lane & 7));
    last = (uint32_t)((lane >> 3) * rb + 16 * (lane & 3));
    z = 4 * (lane & 15);
    rows8 = 8 * rb;
  }
};

template <int NU, int FMT>
__device__ __forceinline__ void load_unit(Unit<FMT>& b, const Source<NU>& src, const Place<FMT>& at, int u, int gr) {
  const bool alone = FMT == FMT_Q4 && gr + 1 == at.ng;
  const uint8_t* const w = src.w[u] + (FMT == FMT_Q4 ? 64 : 128) * gr;
  const uint32_t off = alone ? at.last : at.whole;
#pragma unroll
  for (int i = 0; i < 2; ++i) b.c[i] = *reinterpret_cast<const u32x4*>(w + i * at.rows8 + off);
#pragma unroll
  for (int h = 0; h < STEP<FMT>; ++h) {
    if constexpr (FMT == FMT_Q4)
      b.z[h] = *reinterpret_cast<const uint32_t*>(src.s[u] + (int64_t)(alone ? gr : gr + h) * at.R * 4 + at.z);
    else b.z[h] = src.s[u][gr];
  }
}
template <int NU>
__device__ __forceinline__ void load_values(Values& b, const Source<NU>& src, int gr) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    b.x[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(src.x, src.x_off + 16 * i, gr * 256, 0));
}

// The codes' way through a wave's LDS: 16 rows of 128 bytes, 16-byte word c of row r at
// c ^ (r / 2), so that the 16 rows which a quarter of the fragment read takes are in different banks.
__device__ __forceinline__ int word_at(int r, int c) { return r * 128 + 16 * (c ^ ((r >> 1) & 7)); }

// Eight 4-bit codes -> a fragment register: bf16 128 + q, or fp16 q - 8.  The constants
// sit in registers, which makes one v_and_or of the two operations (GFX9 takes no literal there).
template <int DT>
struct Nibbles {
  uint32_t keep = 0x000F000Fu, top = DT == USAF_BF16 ? 0x43004300u : 0x64006400u;
  __device__ __forceinline__ Nibbles() { asm("" : "+s"(keep), "+v"(top)); }
  __device__ __forceinline__ u32x4 frag(uint32_t w) const {
    u32x4 o;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const uint32_t t = ((w >> (4 * p)) & keep) | top;
      if constexpr (DT == USAF_BF16) {
        o[p] = t;
      } else {
        const f16x2 c = {(f16)-1032.0f, (f16)-1032.0f};
        o[p] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, t) + c);
      }
    }
    return o;
  }
};
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

template <int DT>
__device__ __forceinline__ f32x4 mfma16(const u32x4 a, const u32x4 b, f32x4 c) {
  if constexpr (DT == USAF_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                   0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// One step of NU units: acc[u] += the product of their rows and the tokens; value i of
// lane (r, q) is token row 4 q + i, weight row r.  Meanwhile b's weights are loaded from src,
// groups gr on, and the tokens' values there: 4-bit, v0 and v1 are a step's two groups (`two`:
// it has the second), each loaded behind its last use; 8-bit, v0 is this step's and v1 the
// next one's.  No load carries a condition, or the compiler would have to wait for all of them at every use.
template <int NU, int FMT, int DT>
__device__ __forceinline__ void mul_step(Unit<FMT> (&b)[NU], Values& v0, Values& v1, bool two, const Source<NU>& src,
                                         const Place<FMT>& at, int gr, uint8_t* lds, int lane, const Nibbles<DT>& nib,
                                         f32x4 (&acc)[NU]) {
  const int r = lane & 15, q = lane >> 4;
  uint32_t z[NU][STEP<FMT>];
  __builtin_amdgcn_wave_barrier();  // one wave's LDS operations complete in order
#pragma unroll
  for (int u = 0; u < NU; ++u) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      *reinterpret_cast<u32x4*>(lds + u * UNIT_LDS + word_at(8 * i + (lane >> 3), lane & 7)) = b[u].c[i];
#pragma unroll
    for (int h = 0; h < STEP<FMT>; ++h) z[u][h] = b[u].z[h];
  }
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int u = 0; u < NU; ++u) load_unit<NU, FMT>(b[u], src, at, u, gr);
  if constexpr (FMT == FMT_FP8) load_values<NU>(v1, src, gr);
  __builtin_amdgcn_sched_barrier(0);
  auto word = [&](int u, int c) { return *reinterpret_cast<const u32x4*>(lds + u * UNIT_LDS + word_at(r, c)); };
  if constexpr (FMT == FMT_Q4) {
    const uint32_t one = DT == USAF_BF16 ? 0x3F803F80u : 0x3C003C00u;
    auto group = [&](int h, const Values& v) {
      f32x4 xs = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 4; ++i) xs = mfma16<DT>(v.x[i], u32x4{one, one, one, one}, xs);
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        const u32x4 c = word(u, 4 * h + q);
        f32x4 d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 4; ++i) d = mfma16<DT>(v.x[i], nib.frag(c[i]), d);
        const float sc = f16_bits_to_f32((uint16_t)z[u][h]);
        const float zo = fmaf(DT == USAF_BF16 ? -128.0f : 8.0f, sc, f16_bits_to_f32((uint16_t)(z[u][h] >> 16)));
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[u][i] = fmaf(zo, xs[i], fmaf(sc, d[i], acc[u][i]));
      }
    };
    group(0, v0);
    __builtin_amdgcn_sched_barrier(0);
    load_values<NU>(v0, src, gr);
    __builtin_amdgcn_sched_barrier(0);
    if (two) group(1, v1);
    __builtin_amdgcn_sched_barrier(0);
    load_values<NU>(v1, src, gr + 1);
  } else {
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const u32x4 c0 = word(u, 2 * q), c1 = word(u, 2 * q + 1);
      f32x4 d = {0.f, 0.f, 0.f, 0.f};
      d = mfma16<DT>(v0.x[0], frag8<DT>(c0.x, c0.y), d);
      d = mfma16<DT>(v0.x[1], frag8<DT>(c0.z, c0.w), d);
      d = mfma16<DT>(v0.x[2], frag8<DT>(c1.x, c1.y), d);
      d = mfma16<DT>(v0.x[3], frag8<DT>(c1.z, c1.w), d);
      const float sc = __uint_as_float(z[u][0] == 0 ? 0x00400000u : z[u][0] << 23);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[u][i] = fmaf(sc, d[i], acc[u][i]);
    }
  }
  __builtin_amdgcn_sched_barrier(0);
}

// An item's tokens as rows of the operand.  Rows past the last are not loaded and their results not used.
struct Tokens {
  int count;   // rows in use
  int own[4];  // tokens of the lane's result rows 4 q + i
  // Returns the lane's operand row's place in a buffer of tokens of `row` bytes.
  __device__ __forceinline__ uint32_t set(const Item& t, int row, int lane) {
    const int r = lane & 15, left = __popc(t.tokens) - FR * t.b;
    count = left > FR ? FR : left;
    const int mine = nth_bit(t.tokens, FR * t.b + (r < count ? r : count - 1));
#pragma unroll
    for (int i = 0; i < 4; ++i) own[i] = __shfl(mine, 4 * (lane >> 4) + i, 64);
    return r < count ? (uint32_t)(mine * row + 64 * (lane >> 4)) : NO_ROW;
  }
};

// Both products walk a list of (item, step) pairs, across the items' ends: a wave has only
// one to eight steps of an item, and a first load takes as long as several steps' arithmetic.
// The last pair's weights are loaded once more.

// Bound by the weights' way from memory where many experts are in use, else by the launch and two trips
// there.  32 gate and their 32 up rows are one item, so that the activation needs no second pass.  Measured
// (weights with scales): 24 tokens, about 101 of 128 experts of 768 x 2,048, 4-bit, 169 MB: 38 us, 4.4 TB/s; 7
// tokens, 8 of 14,336 x 4,096, 4-bit, 433 MB: 85 us, 5.1 TB/s; 32 tokens, 63 of 64 of 1,024 x 2,048, 8-bit,
// 265 MB: 51 us, 5.2 TB/s; one token, 13 MB: 10.6 us with the choice of its experts.
constexpr int GU_NU = 4, GU_WAVES = 4, GU_THREADS = 64 * GU_WAVES;  // 32 gate rows and their 32 up rows

template <int DT, int FMT, bool ROUTES>
__global__ __launch_bounds__(GU_THREADS, 3) void few_gate_up_kernel(const FewArgs g) {
  __shared__ f32x4 red[GU_WAVES][GU_NU][64];
  __shared__ __attribute__((aligned(16))) uint8_t s_codes[GU_WAVES][GU_NU * UNIT_LDS];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int n_nt = g.I / 32, ng = g.H / 128, ns = (ng + STEP<FMT> - 1) / STEP<FMT>;
  const int s0 = ns * wave / GU_WAVES, some = ns * (wave + 1) / GU_WAVES - s0;  // the wave's steps
  const int n = some > 0 ? some : 1;  // a wave without a step of its own multiplies one and adds nothing
  const int first = STEP<FMT> * (s0 < ns ? s0 : ns - 1);
  InUse in;
  if constexpr (ROUTES) {
    // every wave chooses the experts for itself; the first keeps weights and masks for few_down
#pragma unroll
    for (int i = 0; i < InUse::N; ++i) in.mask[i] = 0;
    for (int t = 0; t < g.T; ++t) {
      const Chosen c(g.logits + (int64_t)t * g.E, g.E, g.k, lane);
      if (blockIdx.x == 0 && wave == 0) c.weights(g, t, lane, reinterpret_cast<float*>(&red[0][0][0]));
#pragma unroll
      for (int i = 0; i < InUse::N; ++i) in.mask[i] |= c.rank[i] >= 0 ? 1u << t : 0u;
    }
    if (blockIdx.x == 0 && wave == 0)
#pragma unroll
      for (int i = 0; i < InUse::N; ++i) g.mask[64 * i + lane] = in.mask[i];
    in.find();
  } else {
    in.load(g.mask, lane);
  }
  const int work = in.items * n_nt;
  int at = blockIdx.x, st = 0;  // the pair being loaded
  if (at >= work) return;       // block-uniform
  const Place<FMT> place(2 * g.I, g.H, lane);
  Source<GU_NU> src;
  src.x = buffer_of(FMT == FMT_Q4 ? g.xp : g.x, g.T * g.H * 2);
  auto source = [&]() {
    const Item t = in.item(at / n_nt);
    const int n0 = at % n_nt * 32;
    src.template weights<FMT>(g.gu, g.gu_s, t.e, 2 * g.I, g.H, {n0, n0 + 16, g.I + n0, g.I + n0 + 16});
    Tokens tk;
    src.x_off = tk.set(t, 2 * g.H, lane);
  };
  const Nibbles<DT> nib;
  f32x4 acc[GU_NU];
  auto finish = [&](int done) {
    lds_barrier();  // the last item's sums have been read
#pragma unroll
    for (int v = 0; v < GU_NU; ++v) red[wave][v][lane] = some > 0 ? acc[v] : f32x4{0.f, 0.f, 0.f, 0.f};
    lds_barrier();
    const Item t = in.item(done / n_nt);
    Tokens tk;
    tk.set(t, 2 * g.H, lane);
    // wave: columns n0 + 16 (wave % 2) + [0, 16), two of the lane's four rows
    const int v = wave & 1, j0 = wave & 2;
    const int col = frag_pos<FMT>(done % n_nt * 32 + 16 * v + r);
    f32x4 gt = red[0][v][lane], up = red[0][2 + v][lane];
#pragma unroll
    for (int i = 1; i < GU_WAVES; ++i) {
      const f32x4 a = red[i][v][lane], c = red[i][2 + v][lane];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        gt[j] += a[j];
        up[j] += c[j];
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float gv = j0 ? gt[2 + j] : gt[j], uv = j0 ? up[2 + j] : up[j];
      const int tok = j0 ? tk.own[2 + j] : tk.own[j];
      if (4 * q + j0 + j < tk.count)
        store_from_f32<DT>(g.act, ((int64_t)t.u * g.T + tok) * g.I + col, silu_fast(gv) * uv);
    }
  };
  auto clear = [&]() {
#pragma unroll
    for (int v = 0; v < GU_NU; ++v) acc[v] = f32x4{0.f, 0.f, 0.f, 0.f};
  };
  Unit<FMT> weights[GU_NU];
  Values v0, v1;
  auto step = [&](Values& v0, Values& v1) {  // false: it was the last
    const int done = at, gr = first + STEP<FMT> * st;  // the pair being multiplied
    const bool ends = st == n - 1;
    if (!ends) {
      ++st;
    } else if (at + (int)gridDim.x < work) {
      at += gridDim.x;
      st = 0;
      source();
    }
    mul_step<GU_NU, FMT, DT>(weights, v0, v1, gr + 1 < ng, src, place, first + STEP<FMT> * st, s_codes[wave], lane, nib, acc);
    if (ends) {
      finish(done);
      clear();
      return done + (int)gridDim.x < work;
    }
    return true;
  };
  source();
  clear();
#pragma unroll
  for (int u = 0; u < GU_NU; ++u) load_unit<GU_NU, FMT>(weights[u], src, place, u, first);
  load_values<GU_NU>(v0, src, first);
  if constexpr (FMT == FMT_Q4) {
    load_values<GU_NU>(v1, src, first + 1);
    while (step(v0, v1)) {
    }
  } else {
    while (step(v0, v1) && step(v1, v0)) {
    }
  }
}

// The same bound and, for few pairs, the parts' meeting.  Measured as above: 84 MB 27 us, 3.1 TB/s; 216 MB 48 us, 4.5
// TB/s; 132 MB 33 us, 4.0 TB/s; one token, 7 MB, 8.5 us.  Blocks of 12 waves and 32 columns, which need
// no parts, were 0.3 us quicker for one token on 4-bit experts of 768 and up to 20 us slower elsewhere.
constexpr int DN_WAVES = 4, DN_THREADS = 64 * DN_WAVES, DN_NU = 4, DN_COLS = 16 * DN_NU;

template <int DT, int FMT>
__global__ __launch_bounds__(DN_THREADS) void few_down_kernel(const FewArgs g) {
  // the waves' codes, and their sums [waves][T][64]: 64 KiB at most
  extern __shared__ __attribute__((aligned(16))) uint8_t s_down[];
  float* const s_sum = reinterpret_cast<float*>(s_down + DN_WAVES * DN_NU * UNIT_LDS);
  int* const s_last = reinterpret_cast<int*>(s_down);  // once the codes have been read
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int nt = blockIdx.x / g.P, p = blockIdx.x - nt * g.P, n0 = DN_COLS * nt;
  float* const sum = s_sum + wave * g.T * DN_COLS;  // the wave's own: its LDS operations complete in order
  uint8_t* const codes = s_down + wave * DN_NU * UNIT_LDS;
  for (int i = lane; i < g.T * DN_COLS / 4; i += 64) reinterpret_cast<f32x4*>(sum)[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  InUse in;
  in.load(g.mask, lane);
  // the wave's pairs: an even share of all waves' of this column tile
  const int ng = g.I / 128, ns = (ng + STEP<FMT> - 1) / STEP<FMT>, work = in.items * ns, parts = g.P * DN_WAVES;
  const int part = p * DN_WAVES + wave;
  const int f1 = (int)((int64_t)work * (part + 1) / parts);
  int f = (int)((int64_t)work * part / parts);  // the pair being loaded
  if (f < f1) {
    int it = f / ns, st = f - it * ns;
    const Place<FMT> place(g.H, g.I, lane);
    Source<DN_NU> src;
    Tokens tk, next_tk;
    float wt[4], next_wt[4];
    auto source = [&]() {
      const Item t = in.item(it);
      src.template weights<FMT>(g.dn, g.dn_s, t.e, g.H, g.I, {n0, n0 + 16, n0 + 32, n0 + 48});
      src.x = buffer_of(g.act + (int64_t)t.u * g.T * g.I, g.T * g.I * 2);
      src.x_off = next_tk.set(t, 2 * g.I, lane);
#pragma unroll
      for (int i = 0; i < 4; ++i) next_wt[i] = g.wt[t.e * FT + next_tk.own[i]];
    };
    const Nibbles<DT> nib;
    f32x4 y[DN_NU];
    auto begin = [&]() {
      tk = next_tk;
#pragma unroll
      for (int i = 0; i < 4; ++i) wt[i] = next_wt[i];
#pragma unroll
      for (int v = 0; v < DN_NU; ++v) y[v] = f32x4{0.f, 0.f, 0.f, 0.f};
    };
    Unit<FMT> weights[DN_NU];
    Values v0, v1;
    auto step = [&](Values& v0, Values& v1) {
      const int gr = STEP<FMT> * st;
      bool ends = true;
      if (++f < f1) {
        if (++st == ns) {
          st = 0;
          ++it;
          source();
        } else {
          ends = false;
        }
      }
      mul_step<DN_NU, FMT, DT>(weights, v0, v1, gr + 1 < ng, src, place, STEP<FMT> * st, codes, lane, nib, y);
      if (ends) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (4 * q + i < tk.count) {
#pragma unroll
            for (int v = 0; v < DN_NU; ++v) {
              float* const to = sum + tk.own[i] * DN_COLS + 16 * v + r;
              *to = fmaf(wt[i], y[v][i], *to);
            }
          }
        __builtin_amdgcn_wave_barrier();
        begin();
      }
      return f < f1;
    };
    source();
    begin();
#pragma unroll
    for (int u = 0; u < DN_NU; ++u) load_unit<DN_NU, FMT>(weights[u], src, place, u, STEP<FMT> * st);
    load_values<DN_NU>(v0, src, STEP<FMT> * st);
    if constexpr (FMT == FMT_Q4) {
      load_values<DN_NU>(v1, src, STEP<FMT> * st + 1);
      while (step(v0, v1)) {
      }
    } else {
      while (step(v0, v1) && step(v1, v0)) {
      }
    }
  }
  __syncthreads();
  // four columns of a token at a time
  const int quads = g.T * (DN_COLS / 4);
  const Buffer part_buf = buffer_of(g.part + (int64_t)p * g.T * g.H, g.T * g.H * 4);
  auto place = [&](int i) { return (i / (DN_COLS / 4)) * g.H + n0 + i % (DN_COLS / 4) * 4; };
  auto store_out = [&](int at, f32x4 v) {
    *reinterpret_cast<uint2*>(g.out + at) = uint2{pack2<DT>(v.x, v.y), pack2<DT>(v.z, v.w)};
  };
  for (int i = tid; i < quads; i += DN_THREADS) {
    f32x4 v = reinterpret_cast<const f32x4*>(s_sum)[i];
#pragma unroll
    for (int j = 1; j < DN_WAVES; ++j) {
      const f32x4 o = reinterpret_cast<const f32x4*>(s_sum)[j * quads + i];
#pragma unroll
      for (int c = 0; c < 4; ++c) v[c] += o[c];
    }
    if (g.P == 1) store_out(place(i), v);
    else __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), part_buf, place(i) * 4, 0, DEVICE_SCOPE);
  }
  if (g.P == 1) return;
  // The parts of a column tile meet at the device's coherence point: stored and loaded at
  // device scope, which passes the dies' L2s, and counted behind a wait for the stores.  The
  // last block adds them in order, so the sum does not hang on who came last; no block waits for another.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0)
    *s_last = __hip_atomic_fetch_add(&g.done[nt], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == g.P - 1;
  __syncthreads();
  if (!*s_last) return;
  const Buffer all = buffer_of(g.part, g.P * g.T * g.H * 4);
  for (int i = tid; i < quads; i += DN_THREADS) {
    const int at = place(i);
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int j = 0; j < g.P; j += 4) {
      f32x4 v[4];  // parts past the last read as zeros
#pragma unroll
      for (int k = 0; k < 4; ++k)
        v[k] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(all, (uint32_t)(((j + k) * g.T * g.H + at) * 4),
                                                                               0, DEVICE_SCOPE));
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[c] += v[k][c];
    }
    store_out(at, o);
  }
}

struct FewPlan {
  int64_t in_use, logits, mask, wt, xp, act, part, done, bytes;
  int P;
};

// Sizes, and where each buffer sits in the workspace (16-byte steps).
FewPlan few_plan(int64_t T, int64_t E, int64_t k, int64_t H, int64_t I, bool eight_bit) {
  FewPlan p;
  p.in_use = E < T * k ? E : T * k;
  // two blocks a CU for the column tiles together, and about two pairs a wave at least (which 8-bit codes have
  // more of: their plan never takes less of the workspace)
  const int64_t tiles = H / DN_COLS, cus = device_cu_count(), pairs = p.in_use * (I / 128) / (eight_bit ? 1 : 2);
  int64_t parts = 2 * cus / tiles, most = pairs / (2 * DN_WAVES);
  parts = parts > most ? most : parts;
  p.P = (int)(parts < 1 ? 1 : parts);
  int64_t at = 0;
  auto take = [&](int64_t bytes) { const int64_t b = at; at += (bytes + 15) / 16 * 16; return b; };
  p.logits = take(T * E * 8);
  p.mask = take(F_MAX_E * 4);
  p.wt = take(E * FT * 4);
  p.done = take(tiles * 4);
  p.xp = take(T * H * 2);
  p.act = take(p.in_use * T * I * 2);
  p.part = take(p.P > 1 ? p.P * T * H * 4 : 0);
  p.bytes = at;
  return p;
}

template <int DT, int FMT>
int launch_few_layer(const FewArgs& g, int64_t in_use, hipStream_t st) {
  if (g.T == 1) few_logits_kernel<DT, FMT, 1><<<(unsigned)g.E, 256, 0, st>>>(g);
  else few_logits_kernel<DT, FMT, 4><<<(unsigned)(g.E * ((g.T + 3) / 4)), 256, 0, st>>>(g);
  if (int rc = check_launch("moe_few/logits")) return rc;
  // Every wave of few_gate_up chooses one or two tokens' experts itself, which saves a launch; more tokens, one
  // behind the other there, take longer than few_route's blocks.  Measured (us, the whole layer, there / with
  // few_route): one token 21.5 / 22.9 (128 experts of 768, 4-bit), 22.4 / 24.3 (8-bit), 21.2 / 23.1 (64 of 1,024), 50.9 /
  // 52.9 (8 of 14,336); two 28.4 / 28.6, 31.9 / 32.0, 28.7 / 29.1; three 35.6 / 34.1, 41.2 / 39.1, 36.1 / 34.6.
  const bool routes = g.T <= 2;
  if (!routes) {
    few_route_kernel<<<(unsigned)g.T, 64, 0, st>>>(g);
    if (int rc = check_launch("moe_few/route")) return rc;
  }
  const int64_t most = 3 * (int64_t)device_cu_count(), work = (in_use + g.T * g.k / (FR + 1)) * (g.I / 32);
  const unsigned blocks = (unsigned)(work < most ? work : most);
  if (routes) few_gate_up_kernel<DT, FMT, true><<<blocks, GU_THREADS, 0, st>>>(g);
  else few_gate_up_kernel<DT, FMT, false><<<blocks, GU_THREADS, 0, st>>>(g);
  if (int rc = check_launch("moe_few/gate_up")) return rc;
  few_down_kernel<DT, FMT>
      <<<(unsigned)(g.H / DN_COLS * g.P), DN_THREADS,
         (size_t)DN_WAVES * (DN_NU * UNIT_LDS + g.T * DN_COLS * 4), st>>>(g);
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
  return T == 0 ? 0 : few_plan(T, E, top_k, H, I, true).bytes;
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
  if ((!eight_bit && ((uintptr_t)gate_up_scale | (uintptr_t)down_scale) % 4) || (uintptr_t)out % 8)
    return set_error(USAF_ERR_INVALID, "moe_few: misaligned scales or output (8 bytes)");
  const FewPlan p = few_plan(T, E, top_k, H, I, eight_bit != 0);
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
  g.logits = reinterpret_cast<double*>(b + p.logits);
  g.mask = reinterpret_cast<uint32_t*>(b + p.mask);
  g.wt = reinterpret_cast<float*>(b + p.wt);
  g.done = reinterpret_cast<int32_t*>(b + p.done);
  g.xp = reinterpret_cast<uint16_t*>(b + p.xp);
  g.act = reinterpret_cast<uint16_t*>(b + p.act);
  g.part = reinterpret_cast<float*>(b + p.part);
  g.P = p.P;
  hipStream_t st = as_stream(stream);
  if (eight_bit)
    return dtype == USAF_BF16 ? launch_few_layer<USAF_BF16, FMT_FP8>(g, p.in_use, st)
                              : launch_few_layer<USAF_F16, FMT_FP8>(g, p.in_use, st);
  return dtype == USAF_BF16 ? launch_few_layer<USAF_BF16, FMT_Q4>(g, p.in_use, st)
                            : launch_few_layer<USAF_F16, FMT_Q4>(g, p.in_use, st);
}

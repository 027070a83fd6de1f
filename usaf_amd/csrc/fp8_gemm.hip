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
//
// A block of eight waves has a tile of 32 MW MI slots x 32 NW NI columns.  Both operands
// come by LDS DMA, one 128-byte line of each row a step, into a ring of NS stages; at a
// step's one barrier its stage has landed and the stage before it has been read, so the
// DMAs of the step NS - 1 ahead go there.  16-byte chunks of a row are XOR-swizzled by
// the row (by the DMA's source address), which makes the fragment reads free of bank conflicts.
#include "fp8.h"

namespace usaf {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void* lds_void_ptr;

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
  int n_nt;
};

constexpr int G_WAVES = 8, G_THREADS = 64 * G_WAVES;
constexpr int G_XCDS = 8;  // accelerator dies, blocks dispatched round-robin over them

__device__ __forceinline__ int g_swz(int r) { return (r >> 1) & 7; }

__device__ __forceinline__ f32x16 mfma8(const u32x4 a0, const u32x4 a1, const u32x4 b0, const u32x4 b1, f32x16 c, int sa,
                                        int sb) {
  const i32x8 a = {(int)a0.x, (int)a0.y, (int)a0.z, (int)a0.w, (int)a1.x, (int)a1.y, (int)a1.z, (int)a1.w};
  const i32x8 b = {(int)b0.x, (int)b0.y, (int)b0.z, (int)b0.w, (int)b1.x, (int)b1.y, (int)b1.z, (int)b1.w};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, 0, sa, 0, sb);
}

// LDS DMA: lane l's 16 (4) bytes at base + off land at lds + 16 l (4 l); base and lds are
// wave-uniform.  Inline asm, since beside the compiler's own LDS DMA every LDS read would
// wait for all of them.  M0 takes the LDS address; the wait states cover a base that comes
// out of readfirstlane.  They count in vmcnt only, which the ring waits for itself.
__device__ __forceinline__ void g_dma16(const void* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "m0");
}
__device__ __forceinline__ void g_dma4(const void* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dword %1, %2" ::"s"(lds), "v"(off), "s"(base) : "m0");
}
__device__ __forceinline__ const uint8_t* uniform(const uint8_t* p) {
  const uint64_t v = (uint64_t)(uintptr_t)p;
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(v >> 32));
  return reinterpret_cast<const uint8_t*>((uintptr_t)(((uint64_t)hi << 32) | (uint64_t)lo));
}
template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Tiles of all experts (one wave, offsets from global memory; E <= 255).
template <int SLOTS>
__device__ __forceinline__ int all_tiles(const int32_t* offsets, int E, int lane) {
  int n = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int i = 4 * lane + k;
    if (i < E) n += (offsets[i + 1] - offsets[i] + SLOTS - 1) / SLOTS;
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) n += __shfl_xor(n, d, 64);
  return __builtin_amdgcn_readfirstlane(n);
}

template <int MW, int MI, int NI>
struct Tile {
  static constexpr int NW = G_WAVES / MW;
  static constexpr int M = 32 * MW * MI, N = 32 * NW * NI;
  static constexpr int A_BYTES = M * 128, W_BYTES = N * 128;
  static constexpr int A_SCALES = M < 64 ? 256 : 4 * M;  // a word for each slot, 64 at a time
  static constexpr int STAGE = A_BYTES + W_BYTES + A_SCALES + 256;  // and 64 words of the weight's
  static constexpr int FIT = 160 * 1024 / STAGE, NS = FIT > 4 ? 4 : FIT;
  static constexpr int LDS = NS * STAGE;
  static constexpr int A_DMA = M >= 64 ? M / 64 : 1, W_DMA = N / 64, DMAS = A_DMA + W_DMA + 1;
  static constexpr int OUT_ROW = 64 * NI;  // bytes of a wave's row of results
  static_assert(NS >= 2 && M <= 256 && G_WAVES * 32 * MI * OUT_ROW <= LDS, "LDS");
};

template <int MW, int MI, int NI, int DT>
__global__ __launch_bounds__(G_THREADS) void fp8_gemm_kernel(const Fp8Args g) {
  typedef Tile<MW, MI, NI> T;
  extern __shared__ __attribute__((aligned(16))) uint8_t sm[];
  const uint32_t sm_lds = (uint32_t)(uintptr_t)(lds_void_ptr)sm;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, half = lane >> 5;
  const int wm = wave % MW, wn = wave / MW;

  // ---- the block's tile.  A die's blocks take a run of the list, so that what they share sits
  //      in its L2: of one expert, or of one weight, eight slot tiles side by side
  const int m_tiles = g.offsets ? all_tiles<T::M>(g.offsets, g.E, lane) : (int)((g.M + T::M - 1) / T::M);
  const int tiles = m_tiles * g.n_nt, per = (tiles + G_XCDS - 1) / G_XCDS;
  const int j = (int)blockIdx.x / G_XCDS, id = ((int)blockIdx.x % G_XCDS) * per + j;
  if (j >= per || id >= tiles) return;  // block-uniform
  int mt, nt, e = 0, valid;
  int64_t m_beg;
  if (g.offsets) {
    mt = id / g.n_nt;
    nt = id - mt * g.n_nt;
    GemmArgs o{};
    o.offsets = g.offsets;
    o.E = g.E;
    int beg;
    if (!slot_tile<T::M>(o, lane, mt, e, beg, valid)) return;
    m_beg = beg;
  } else {
    constexpr int GROUP = 8;
    const int band = id / (GROUP * g.n_nt), rest = id - band * GROUP * g.n_nt;
    const int tall = m_tiles - band * GROUP < GROUP ? m_tiles - band * GROUP : GROUP;
    nt = rest / tall;
    mt = band * GROUP + rest - nt * tall;
    m_beg = (int64_t)mt * T::M;
    valid = g.M - m_beg < T::M ? (int)(g.M - m_beg) : T::M;
  }
  const int64_t n0 = (int64_t)nt * T::N;
  const int nkb = (int)(g.Kp / 128);

  // ---- DMA sources: uniform bases, 32-bit lane offsets.  Instruction i of wave w fills rows
  //      8 (8 i + w) + [0, 8) of the stage, lane l chunk l % 8 of row l / 8
  const uint8_t* a_base = uniform(g.a_rows ? g.A : g.A + m_beg * g.Kp);
  const uint8_t* w_base = uniform(g.W + ((int64_t)e * g.N + n0) * g.Kp);
  auto slot_row = [&](int r) -> int64_t {  // operand row of slot r of the tile, from a_base's
    r = r < valid ? r : valid - 1;
    return g.a_rows ? (int64_t)g.a_rows[m_beg + r] : r;
  };
  uint32_t a_off[T::A_DMA], w_off[T::W_DMA];
#pragma unroll
  for (int i = 0; i < T::A_DMA; ++i) {
    const int r = (8 * (8 * i + wave) + (lane >> 3)) % T::M;  // (tiles of 32 slots: two waves fill each row)
    a_off[i] = (uint32_t)(slot_row(r) * g.Kp) + 16 * ((lane & 7) ^ g_swz(r));
  }
#pragma unroll
  for (int i = 0; i < T::W_DMA; ++i) {
    const int r = 8 * (8 * i + wave) + (lane >> 3);
    const int64_t n = n0 + r < g.N ? r : g.N - 1 - n0;
    w_off[i] = (uint32_t)(n * g.Kp) + 16 * ((lane & 7) ^ g_swz(r));
  }
  // scales, a word for each row: waves below M / 64 those of 64 slots each, the others (all the
  // same) those of the tile's blocks of 128 columns, the words around the byte
  constexpr int A_SCALE_WAVES = (T::M + 63) / 64;
  const bool a_scale = wave < A_SCALE_WAVES;
  const uint8_t* const s_base = uniform(a_scale ? (g.a_rows ? g.as : g.as + m_beg * g.sp) : g.ws);
  const int64_t nrb = (g.N + 127) / 128;
  const int ws_shift = (int)((uintptr_t)g.ws & 3);
  int64_t ws_row = (n0 / 128 + (lane < 2 ? lane : 0));
  ws_row = ((int64_t)e * nrb + (ws_row < nrb ? ws_row : nrb - 1)) * nkb + ws_shift;
  const uint32_t s_off = a_scale ? (uint32_t)(slot_row((64 * wave + lane) % T::M) * g.sp) : 0;
  const uint32_t s_lds = (uint32_t)(T::A_BYTES + T::W_BYTES + (a_scale ? 256 * wave : T::A_SCALES));

  auto issue = [&](int kb, int stage) {
    kb = kb < nkb ? kb : nkb - 1;
    const uint32_t to = (uint32_t)__builtin_amdgcn_readfirstlane((int)(sm_lds + stage * T::STAGE));
    const uint8_t* const a = a_base + (int64_t)kb * 128;
    const uint8_t* const w = w_base + (int64_t)kb * 128;
#pragma unroll
    for (int i = 0; i < T::A_DMA; ++i) g_dma16(a, a_off[i], to + (8 * i + wave) * 1024 % T::A_BYTES);
#pragma unroll
    for (int i = 0; i < T::W_DMA; ++i) g_dma16(w, w_off[i], to + T::A_BYTES + (8 * i + wave) * 1024);
    if (a_scale) g_dma4(s_base + (kb & ~3), s_off, to + s_lds);
    else g_dma4(s_base - ws_shift, (uint32_t)((ws_row + kb) & ~(int64_t)3), to + s_lds);
  };

  f32x16 acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int k = 0; k < NI; ++k) acc[i][k] = f32x16{};
  const int mine = valid - 32 * MI * wm;  // slots of the wave's part
  const int live = mine <= 0 ? 0 : mine >= 32 * MI ? MI : (mine + 31) >> 5;  // its blocks of 32 with any

  for (int s = 0; s < T::NS - 1; ++s) issue(s, s);
  int stage = 0;
  for (int kb = 0; kb < nkb; ++kb) {
    wait_vmcnt<(T::NS - 2) * T::DMAS>();  // the wave's DMAs of this step
    lds_barrier();                        // and everyone's; the stage before this one has been read
    issue(kb + T::NS - 1, stage == 0 ? T::NS - 1 : stage - 1);
    const uint8_t* const sa = sm + stage * T::STAGE;
    const uint8_t* const sw = sa + T::A_BYTES;
    const uint32_t* const sc = reinterpret_cast<const uint32_t*>(sw + T::W_BYTES);
    auto word = [&](const uint8_t* rows, int r, int c) {
      return *reinterpret_cast<const u32x4*>(rows + r * 128 + 16 * (c ^ g_swz(r)));
    };
    int s_a[MI], s_w[NI];
#pragma unroll
    for (int i = 0; i < MI; ++i) s_a[i] = (int)(sc[32 * (MI * wm + i) + l32] >> (8 * (kb & 3)));
#pragma unroll
    for (int k = 0; k < NI; ++k) {
      const int b = (32 * (NI * wn + k)) / 128;  // which block of 128 columns
      int64_t at = n0 / 128 + b;
      at = ((int64_t)e * nrb + (at < nrb ? at : nrb - 1)) * nkb + ws_shift + kb;
      s_w[k] = (int)(sc[T::A_SCALES / 4 + b] >> (8 * (int)(at & 3)));
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = 4 * h + 2 * half;
      u32x4 w0[NI], w1[NI];
#pragma unroll
      for (int k = 0; k < NI; ++k) {
        w0[k] = word(sw, 32 * (NI * wn + k) + l32, c);
        w1[k] = word(sw, 32 * (NI * wn + k) + l32, c + 1);
      }
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        if (i >= live) continue;  // wave-uniform
        const u32x4 a0 = word(sa, 32 * (MI * wm + i) + l32, c), a1 = word(sa, 32 * (MI * wm + i) + l32, c + 1);
#pragma unroll
        for (int k = 0; k < NI; ++k) acc[i][k] = mfma8(w0[k], w1[k], a0, a1, acc[i][k], s_w[k], s_a[i]);
      }
    }
    stage = stage + 1 == T::NS ? 0 : stage + 1;
  }
  wait_vmcnt<0>();
  lds_barrier();  // no DMA is under way, nobody reads the ring

  // ---- results: lane's values 4 q .. 4 q + 3 of a 32 x 32 block are columns 8 q + 4 half +
  //      [0, 4) of slot l32.  Through the wave's part of LDS, for whole lines to memory
  uint8_t* const so = sm + wave * (32 * MI * T::OUT_ROW);
  constexpr int CH = T::OUT_ROW / 16;  // 16-byte chunks of a row
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int k = 0; k < NI; ++k)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int r = 32 * i + l32, c = 4 * k + q;
        *reinterpret_cast<uint2*>(so + r * T::OUT_ROW + 16 * (c ^ (r & (CH - 1))) + 8 * half) =
            uint2{pack2<DT>(acc[i][k][4 * q], acc[i][k][4 * q + 1]), pack2<DT>(acc[i][k][4 * q + 2], acc[i][k][4 * q + 3])};
      }
  __builtin_amdgcn_wave_barrier();
  const bool wide = g.N % 8 == 0 && ((uintptr_t)g.out & 15) == 0;
  const int64_t nw = n0 + 32 * NI * wn;
#pragma unroll 4
  for (int it = 0; it < 32 * MI * CH / 64; ++it) {
    const int r = it * (64 / CH) + lane / CH, c = lane % CH;
    const u32x4 v = *reinterpret_cast<const u32x4*>(so + r * T::OUT_ROW + 16 * (c ^ (r & (CH - 1))));
    const int64_t n = nw + 8 * c;
    if (r >= mine || n >= g.N) continue;
    uint16_t* const to = g.out + (m_beg + 32 * MI * wm + r) * g.N + n;
    if (wide) {
      *reinterpret_cast<u32x4*>(to) = v;
    } else {
#pragma unroll
      for (int b = 0; b < 8; ++b)
        if (n + b < g.N) to[b] = (uint16_t)(v[b >> 1] >> (16 * (b & 1)));
    }
  }
}

bool raise_fp8_lds(const void* kernel, size_t bytes) {
  (void)hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  (void)hipGetLastError();
  return true;
}
template <int MW, int MI, int NI, int DT>
void prepare_one() {
  static const bool done = raise_fp8_lds(reinterpret_cast<const void*>(&fp8_gemm_kernel<MW, MI, NI, DT>),
                                         Tile<MW, MI, NI>::LDS);
  (void)done;
}

template <int MW, int MI, int NI>
int launch(Fp8Args g, int dt, hipStream_t st) {
  typedef Tile<MW, MI, NI> T;
  const int64_t m_tiles = g.offsets ? (g.M < g.E ? g.M : g.E) + g.M / T::M : (g.M + T::M - 1) / T::M;
  const int64_t n_nt = (g.N + T::N - 1) / T::N, blocks = (m_tiles * n_nt + G_XCDS - 1) / G_XCDS * G_XCDS;
  if (blocks >= (int64_t)1 << 31) return set_error(USAF_ERR_INVALID, "fp8_gemm: too many tiles");
  g.n_nt = (int)n_nt;
  if (dt == USAF_BF16) {
    prepare_one<MW, MI, NI, USAF_BF16>();
    fp8_gemm_kernel<MW, MI, NI, USAF_BF16><<<(unsigned)blocks, G_THREADS, T::LDS, st>>>(g);
  } else {
    prepare_one<MW, MI, NI, USAF_F16>();
    fp8_gemm_kernel<MW, MI, NI, USAF_F16><<<(unsigned)blocks, G_THREADS, T::LDS, st>>>(g);
  }
  return check_launch("fp8_gemm");
}

}  // namespace

void prepare_fp8_kernels() {
  prepare_one<1, 1, 1, USAF_BF16>();
  prepare_one<1, 1, 1, USAF_F16>();
  prepare_one<1, 2, 1, USAF_BF16>();
  prepare_one<1, 2, 1, USAF_F16>();
  prepare_one<2, 2, 2, USAF_BF16>();
  prepare_one<2, 2, 2, USAF_F16>();
  prepare_one<2, 4, 2, USAF_BF16>();
  prepare_one<2, 4, 2, USAF_F16>();
}

}  // namespace usaf

using namespace usaf;

extern "C" int usaf_hip_fp8_gemm(const uint8_t* a, const uint8_t* a_scale, int64_t a_total, const int32_t* a_rows, int64_t M,
                                 const uint8_t* w, const uint8_t* w_scale, const int32_t* offsets, int64_t E, int64_t N,
                                 int64_t K, int32_t dtype, void* out, void* stream) {
  if (M < 0 || N < 0 || K < 0 || E < 1 || N > 1 << 24 || K > 1 << 24 || M > 0x7FFFFFFF || a_total < 0)
    return set_error(USAF_ERR_INVALID, "fp8_gemm: bad size M=%lld N=%lld K=%lld E=%lld", (long long)M, (long long)N,
                     (long long)K, (long long)E);
  if (dtype != USAF_BF16 && dtype != USAF_F16) return set_error(USAF_ERR_INVALID, "fp8_gemm: dtype must be fp16 or bf16");
  if (M == 0 || N == 0) return clear_error();
  if (K == 0) return set_error(USAF_ERR_INVALID, "fp8_gemm: need K >= 1");
  if (!a || !a_scale || !w || !w_scale || !out) return set_error(USAF_ERR_INVALID, "fp8_gemm: null pointer");
  if (!offsets && E != 1) return set_error(USAF_ERR_INVALID, "fp8_gemm: more than one expert needs offsets");
  if (!a_rows && M > a_total) return set_error(USAF_ERR_INVALID, "fp8_gemm: more slots than rows");
  if (E > Q_MAX_E) return set_error(USAF_ERR_UNSUPPORTED, "fp8_gemm: at most %d experts", Q_MAX_E);
  if (((uintptr_t)a | (uintptr_t)w) % 16 || (uintptr_t)a_scale % 4 || (uintptr_t)out % 2)
    return set_error(USAF_ERR_INVALID, "fp8_gemm: codes must be 16-byte, scales 4-byte and the output 2-byte aligned");
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
  // 32-bit offsets: gathered rows, a tile of 256 rows of either operand, the weight's scales
  if ((a_rows && a_total * g.Kp >= (int64_t)1 << 32) || 256 * g.Kp >= (int64_t)1 << 32 ||
      E * ((N + 127) / 128) * (g.Kp / 128) >= (int64_t)1 << 31)
    return set_error(USAF_ERR_UNSUPPORTED, "fp8_gemm: operands past 4 GiB of gathered rows or 2 GiB of scales");
  hipStream_t st = as_stream(stream);
  const int64_t per = M / E;  // slots of an expert on average
  if (per <= 32) return launch<1, 1, 1>(g, dtype, st);
  if (per <= 64) return launch<1, 2, 1>(g, dtype, st);
  if (per <= 128) return launch<2, 2, 2>(g, dtype, st);
  return launch<2, 4, 2>(g, dtype, st);
}

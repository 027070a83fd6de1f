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
// A block of eight waves has tiles of 32 MW MI slots x 32 NW NI columns; KW of its waves
// split the contraction's blocks.  Blocks stay (one a CU) and walk a die's run of the tile list.
// Both operands come by LDS DMA, 128-byte lines of KW k-blocks a step, into a ring of NS
// stages; at a step's one barrier its stage has landed and the stage before it has been
// read, so the DMAs of the step NS - 1 ahead go there, straight across tile ends: a tile of 6
// steps (a contraction of 768) would spend as long on its first lines as on its products.
// 16-byte chunks of a row are XOR-swizzled by the row (by the DMA's source address), which
// spreads the fragment reads over the banks (conflicts: 3 % of the LDS's cycles).
//
// Sums: the 8-bit instruction aligns the 64 products within it to the largest and cuts what lies below about 2^-13 of it.
// On normal data that is 1.5e-5 of a result (rms): one bf16 result in 80 and one fp16 result in 15 is the neighbour of the
// nearest.  With a column 100 times the others in every 128 it is one in 25 and one in 5, the distance to the exact
// product 1.66e-3 in bf16 as by its rounding alone and 2.19e-4 in fp16 against 2.07e-4; a result that is left of larger
// products which cancel loses more.  WIDE multiplies the same values with the 16-bit instruction, whose sums are fp32's.
//
// Many rows: 8,192 x 14,336 x 4,096 takes 834,000 cycles, the matrix instructions busy 55 % of them, the LDS's reads 26 %;
// a wave waits 34 % of its cycles, for a step's lines and its barrier.  The clock falls from 1.9 to 1.5 GHz under it: 430 us
// the first times, up to 540, 489 on average over 24 passes in a row (2.0 PFLOP/s), 427 with pauses (the library's product of the
// same codes, unscaled: 386 to 398); by the 16-bit instruction 760 to 830 us, 1.2 PFLOP/s, where the library's 16-bit product of these sizes
// reaches 1.4 to 1.5.  For few rows the weights' way from memory: 128 experts' 768 x 2,048 gate and up, 402 MB, with 2 to 16
// slots each, 70 to 75 us, 5.4 TB/s.
//
// ACT: W_e holds a gate's and an up projection's I rows each; a tile is 128 columns of both (each
// wave 32 of one and the same 32 of the other), and what leaves it is only the next product's operand,
// a block of 128 of every slot:  q, s = Q(dt(dt(silu(g)) u)),  with (g, u) = C.  A layer of 2,048
// tokens on 64 experts of 1,024 takes 310 us so and 322 with C written and a kernel of its own behind it.  Where a
// backward needs C as well the two are equal (846, 4,096 tokens on 128 experts of 768), or this
// one is the slower (352 against 343, 256 tokens), so there they stay apart.
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
  uint16_t* out;           // [M, N]; not ACT
  int n_nt;
  // ACT: N = 2 I
  uint8_t* q;              // [M, I] codes of the gated activation
  uint8_t* qs;             // [M, q_sp] their scale bytes
  int q_sp;
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

// The list of m-tiles (experts in order, each in tiles of SLOTS), held by a wave: lane l
// has experts 4 l .. 4 l + 3 (E <= 255).
template <int SLOTS>
struct SlotTiles {
  int off[5], c[4], incl, sum, total;
  __device__ __forceinline__ void load(const int32_t* offsets, int E, int lane) {
    sum = 0;
#pragma unroll
    for (int k = 0; k < 5; ++k) off[k] = offsets[4 * lane + k < E ? 4 * lane + k : E];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      c[k] = (off[k + 1] - off[k] + SLOTS - 1) / SLOTS;
      sum += c[k];
    }
    incl = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(incl, d, 64);
      if (lane >= d) incl += o;
    }
    total = __builtin_amdgcn_readlane(incl, 63);
  }
  // m-tile mt < total -> expert, first slot, slots
  __device__ __forceinline__ void tile(int mt, int lane, int& e, int& beg, int& valid) const {
    const int src = __builtin_ctzll(__ballot(incl > mt));
    int j = mt - (incl - sum), ee = 4 * lane, b = off[0], end = off[1];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      if (ee == 4 * lane + k && j >= c[k]) {  // past expert 4 l + k
        j -= c[k];
        ee = 4 * lane + k + 1;
        b = off[k + 1];
        end = off[k + 2];
      }
    }
    e = __builtin_amdgcn_readlane(ee, src);
    beg = __builtin_amdgcn_readlane(b + j * SLOTS, src);
    const int rem = __builtin_amdgcn_readlane(end, src) - beg;
    valid = rem < SLOTS ? rem : SLOTS;
  }
};

template <int MW, int NW, int MI, int NI>
struct Tile {
  static constexpr int KW = G_WAVES / (MW * NW);
  static constexpr int M = 32 * MW * MI, N = 32 * NW * NI;
  static constexpr int A_BYTES = M * 128, W_BYTES = N * 128;         // of one k-block
  static constexpr int SCALES = 4 * 64 * ((M + 63) / 64) + 256;      // a word for each slot, 64 words of the weight's
  static constexpr int SLAB = A_BYTES + W_BYTES + SCALES, STAGE = KW * SLAB;
  static constexpr int FIT = 160 * 1024 / STAGE, NS = FIT > 4 ? 4 : FIT, LDS = NS * STAGE;
  // DMA instructions of a wave and step: the rows of its own k-block, shared by the MW NW waves that have it
  static constexpr int SHARE = MW * NW;
  static constexpr int A_DMA = (M / 8 + SHARE - 1) / SHARE, W_DMA = N / 8 / SHARE;
  static constexpr int A_WORDS = (M + 63) / 64;                      // scale instructions of the slots
  static constexpr int S_DMA = (A_WORDS + 1 + SHARE - 1) / SHARE, DMAS = A_DMA + W_DMA + S_DMA;
  static constexpr int OUT_ROW = 64 * NI;                            // bytes of a wave's row of results
  static_assert(NS >= 2 && MW * NW * KW == G_WAVES && N / 8 % SHARE == 0, "tile");
  static_assert(KW > 1 ? G_WAVES * 4096 * NI <= STAGE : G_WAVES * 32 * OUT_ROW <= STAGE, "results go through a stage");
};

template <int MW, int NW, int MI, int NI, int DT, bool WIDE, bool ACT = false>
__global__ __launch_bounds__(G_THREADS) void fp8_gemm_kernel(const Fp8Args g) {
  typedef Tile<MW, NW, MI, NI> T;
  constexpr int KW = T::KW;
  static_assert(!ACT || (NI == 2 && NW == 4 && KW == 1), "a wave has 32 gate and 32 up columns of a block of 128");
  extern __shared__ __attribute__((aligned(16))) uint8_t sm[];
  const uint32_t sm_lds = (uint32_t)(uintptr_t)(lds_void_ptr)sm;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, half = lane >> 5;
  // Experts' last tiles are often half empty: there a SIMD (waves s and s + 4) gets one wave of each half,
  // so that all four have work (512 tokens on 8 experts, 16-bit instruction: 377 -> 336 us).  Full
  // tiles run 2 % faster the other way.
  const int kw = wave / T::SHARE, part = wave % T::SHARE;
  const int wm = g.offsets ? part / NW : part % MW, wn = g.offsets ? part % NW : part / MW;

  // ---- the block's tiles: its die's run of the list, every blocks-of-a-die-th.  What a die's
  //      blocks share at a time sits in its L2: an expert, or eight slot tiles of one weight
  SlotTiles<T::M> slots;
  int m_tiles = (int)((g.M + T::M - 1) / T::M);
  if (g.offsets) {
    slots.load(g.offsets, g.E, lane);
    m_tiles = slots.total;
  }
  const int tiles = m_tiles * g.n_nt, per = (tiles + G_XCDS - 1) / G_XCDS, stride = (int)gridDim.x / G_XCDS;
  const int xcd = (int)blockIdx.x % G_XCDS, run = xcd * per;
  const int end = run + per < tiles ? run + per : tiles, id0 = run + (int)blockIdx.x / G_XCDS;
  if (id0 >= end) return;  // block-uniform
  struct Place {
    int e, valid, nt;
    int64_t m_beg;
  };
  auto place = [&](int id) {
    Place t;
    t.e = 0;
    if (g.offsets) {
      const int mt = id / g.n_nt;
      t.nt = id - mt * g.n_nt;
      int beg;
      slots.tile(mt, lane, t.e, beg, t.valid);
      t.m_beg = beg;
    } else {
      constexpr int GROUP = 8;
      const int band = id / (GROUP * g.n_nt), rest = id - band * GROUP * g.n_nt;
      const int tall = m_tiles - band * GROUP < GROUP ? m_tiles - band * GROUP : GROUP;
      t.nt = rest / tall;
      t.m_beg = (int64_t)(band * GROUP + rest - t.nt * tall) * T::M;
      t.valid = g.M - t.m_beg < T::M ? (int)(g.M - t.m_beg) : T::M;
    }
    return t;
  };
  const int nkb = (int)(g.Kp / 128), steps = (nkb + KW - 1) / KW;
  const int64_t nrb = (g.N + 127) / 128;
  const int ws_shift = (int)((uintptr_t)g.ws & 3);
  // byte of the scale of columns 128 b + [0, 128) of the tile, k-block 0, from the word that ws sits in
  auto ws_at = [&](const Place& t, int b) {
    int64_t at = ACT ? t.nt + b * (g.N / 256) : (int64_t)t.nt * T::N / 128 + b;
    return ((int64_t)t.e * nrb + (at < nrb ? at : nrb - 1)) * nkb + ws_shift;
  };

  // ---- the DMA stream: uniform bases, 32-bit lane offsets.  Of a k-block's rows, instruction i
  //      of wave `part` fills 8 (SHARE i + part) + [0, 8), lane l chunk l % 8 of row l / 8
  int i_id = id0, i_step = 0, i_stage = 0;
  const uint8_t *a_base, *w_base, *as_base;
  uint32_t a_off[T::A_DMA], w_off[T::W_DMA], s_off[T::S_DMA];
  int64_t ws_off = 0;
  auto open = [&]() {
    const Place t = place(i_id);
    const int64_t n0 = (int64_t)t.nt * (ACT ? 128 : T::N);
    a_base = uniform(g.a_rows ? g.A : g.A + t.m_beg * g.Kp);
    as_base = uniform(g.a_rows ? g.as : g.as + t.m_beg * g.sp);
    w_base = uniform(g.W + ((int64_t)t.e * g.N + n0) * g.Kp);
    auto row = [&](int r) -> int64_t {  // operand row of slot r of the tile, from a_base's
      r = r < t.valid ? r : t.valid - 1;
      return g.a_rows ? (int64_t)g.a_rows[t.m_beg + r] : r;
    };
#pragma unroll
    for (int i = 0; i < T::A_DMA; ++i) {
      const int r = (8 * (T::SHARE * i + part) + (lane >> 3)) % T::M;  // (of few rows, some twice)
      a_off[i] = (uint32_t)(row(r) * g.Kp) + 16 * ((lane & 7) ^ g_swz(r));
    }
#pragma unroll
    for (int i = 0; i < T::W_DMA; ++i) {
      const int r = 8 * (T::SHARE * i + part) + (lane >> 3);
      // (ACT: rows 64 wn + 32 k + [0, 32) of the tile are columns 32 wn + [0, 32) of the gate, k = 0, or of up)
      const int64_t n = ACT ? (r >> 5 & 1) * (g.N / 2) + (r >> 6) * 32 + (r & 31) : n0 + r < g.N ? r : g.N - 1 - n0;
      w_off[i] = (uint32_t)(n * g.Kp) + 16 * ((lane & 7) ^ g_swz(r));
    }
    // scale words: instruction s < A_WORDS those of 64 slots, the others (all the same) the
    // weight's, the words around the bytes of the tile's blocks of 128 columns
#pragma unroll
    for (int i = 0; i < T::S_DMA; ++i) {
      const int w = T::SHARE * i + part;
      s_off[i] = w < T::A_WORDS ? (uint32_t)(row((64 * w + lane) % T::M) * g.sp) : 0;
    }
    ws_off = ws_at(t, lane < T::N / 128 ? lane : 0);
  };
  // One step's DMAs, in T::DMAS pieces: begin, the pieces, advance
  uint32_t i_to = 0;
  int i_k = 0;
  const uint8_t *i_a = nullptr, *i_w = nullptr;
  auto begin = [&]() {
    const int kb = i_step * KW + kw;
    i_k = kb < nkb ? kb : nkb - 1;
    i_to = (uint32_t)__builtin_amdgcn_readfirstlane((int)(sm_lds + i_stage * T::STAGE + kw * T::SLAB));
    i_a = a_base + (int64_t)i_k * 128;
    i_w = w_base + (int64_t)i_k * 128;
  };
  auto piece = [&](int p) {
    if (p < T::W_DMA) {
      g_dma16(i_w, w_off[p < T::W_DMA ? p : 0], i_to + T::A_BYTES + (T::SHARE * p + part) * 1024);
    } else if (p < T::W_DMA + T::A_DMA) {
      const int i = p - T::W_DMA;
      g_dma16(i_a, a_off[i < T::A_DMA ? i : 0], i_to + (T::SHARE * i + part) * 1024 % T::A_BYTES);
    } else if (p < T::DMAS) {
      const int i = p - T::W_DMA - T::A_DMA, s = T::SHARE * i + part;  // wave-uniform
      const uint32_t sc = i_to + T::A_BYTES + T::W_BYTES;
      if (s < T::A_WORDS) g_dma4(as_base + (i_k & ~3), s_off[i < T::S_DMA ? i : 0], sc + 256 * s);
      else g_dma4(g.ws - ws_shift, (uint32_t)((ws_off + i_k) & ~(int64_t)3), sc + 256 * T::A_WORDS);
    }
  };
  auto advance = [&]() {
    i_stage = i_stage + 1 == T::NS ? 0 : i_stage + 1;
    if (++i_step == steps) {
      if (i_id + stride < end) {
        i_id += stride;
        i_step = 0;
        open();
      } else {
        i_step = steps - 1;  // past the block's last step: that one again, which nobody reads
      }
    }
  };

  f32x16 acc[MI][NI];
  int stage = 0;
  open();
  for (int s = 0; s < T::NS - 1; ++s) {
    begin();
#pragma unroll
    for (int p = 0; p < T::DMAS; ++p) piece(p);
    advance();
  }
  for (int id = id0; id < end; id += stride) {
    const Place t = place(id);
    const int mine = t.valid - 32 * MI * wm;  // slots of the wave's part
    const int live = mine <= 0 ? 0 : mine >= 32 * MI ? MI : (mine + 31) >> 5;  // its blocks of 32 with any
    int64_t ws_byte[NI];
#pragma unroll
    for (int k = 0; k < NI; ++k) ws_byte[k] = ws_at(t, ACT ? k : (32 * (NI * wn + k)) / 128);
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int k = 0; k < NI; ++k) acc[i][k] = f32x16{};
    for (int step = 0; step < steps; ++step) {
      wait_vmcnt<(T::NS - 2) * T::DMAS>();  // the wave's DMAs of this step (and what is older)
      lds_barrier();                        // and everyone's; the stage before this one has been read
      begin();
      const int kb = step * KW + kw;
      const uint8_t* const sa = sm + stage * T::STAGE + kw * T::SLAB;
      const uint8_t* const sw = sa + T::A_BYTES;
      const uint32_t* const sc = reinterpret_cast<const uint32_t*>(sw + T::W_BYTES);
      stage = stage + 1 == T::NS ? 0 : stage + 1;
      if (KW > 1 && kb >= nkb) {  // wave-uniform
#pragma unroll
        for (int p = 0; p < T::DMAS; ++p) piece(p);
        advance();
        continue;
      }
      auto word = [&](const uint8_t* rows, int r, int c) {
        return *reinterpret_cast<const u32x4*>(rows + r * 128 + 16 * (c ^ g_swz(r)));
      };
      int s_a[MI], s_w[NI];
#pragma unroll
      for (int i = 0; i < MI; ++i) s_a[i] = (int)(sc[32 * (MI * wm + i) + l32] >> (8 * (kb & 3)));
#pragma unroll
      for (int k = 0; k < NI; ++k)
        s_w[k] = (int)(sc[64 * T::A_WORDS + (ACT ? k : (32 * (NI * wn + k)) / 128)] >> (8 * (int)((ws_byte[k] + kb) & 3)));
      // A wave's DMAs go out PER at a time between its matrix instructions: eight waves sending all of
      // theirs first wait for the address unit (16 cycles each, 1,200 in all) before they multiply
      constexpr int SLOTS = MI > 1 ? MI : 2 * MI - 1, PER = (T::DMAS + SLOTS - 1) / SLOTS > 2 ? (T::DMAS + SLOTS - 1) / SLOTS : 2;
      static_assert((2 * MI - 1) * PER >= T::DMAS, "all pieces of a step go out");
      u32x4 w0[NI], w1[NI], a0, a1;
      auto load_w = [&](int h, u32x4(&x0)[NI], u32x4(&x1)[NI]) {
#pragma unroll
        for (int k = 0; k < NI; ++k) {
          x0[k] = word(sw, 32 * (NI * wn + k) + l32, 4 * h + 2 * half);
          x1[k] = word(sw, 32 * (NI * wn + k) + l32, 4 * h + 2 * half + 1);
        }
      };
      auto load_a = [&](int h, int i, u32x4& x0, u32x4& x1) {
        x0 = word(sa, 32 * (MI * wm + i) + l32, 4 * h + 2 * half);
        x1 = word(sa, 32 * (MI * wm + i) + l32, 4 * h + 2 * half + 1);
      };
      load_w(0, w0, w1);
      load_a(0, 0, a0, a1);
      u32x4 wf[WIDE ? NI : 1][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if constexpr (WIDE) {
#pragma unroll
          for (int k = 0; k < NI; ++k) values16(w0[k], w1[k], s_w[k], wf[k]);
        }
        u32x4 v0[NI], v1[NI];
#pragma unroll
        for (int i = 0; i < MI; ++i) {
          // the next fragments, while these are multiplied
          u32x4 b0 = a0, b1 = a1;
          if (i + 1 < MI) {
            load_a(h, i + 1, b0, b1);
          } else if (h == 0) {
            load_w(1, v0, v1);
            load_a(1, 0, b0, b1);
          }
#pragma unroll
          for (int p = 0; p < PER; ++p) {
            const int at = (h * MI + i - 1) * PER + p;  // none before the first matrix instructions
            if (at >= 0) piece(at);
          }
          if (i < live) {  // wave-uniform
            if constexpr (!WIDE) {
#pragma unroll
              for (int k = 0; k < NI; ++k) acc[i][k] = mfma8(w0[k], w1[k], a0, a1, acc[i][k], s_w[k], s_a[i]);
            } else {
              u32x4 af[4];
              values16(a0, a1, s_a[i], af);
#pragma unroll
              for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int k = 0; k < NI; ++k) acc[i][k] = mfma32<USAF_BF16>(wf[k][j], af[j], acc[i][k]);
            }
          }
          a0 = b0;
          a1 = b1;
          __builtin_amdgcn_sched_barrier(0);
        }
        if (h == 0) {
#pragma unroll
          for (int k = 0; k < NI; ++k) {
            w0[k] = v0[k];
            w1[k] = v1[k];
          }
        }
      }
      advance();
    }
    // ---- results, through the stage that was read last: nothing is sent there before the next
    //      step's barrier.  A lane's values 4 q .. 4 q + 3 of a 32 x 32 block are columns 8 q +
    //      4 half + [0, 4) of slot l32
    lds_barrier();
    uint8_t* const free = sm + (stage == 0 ? T::NS - 1 : stage - 1) * T::STAGE;
    const int64_t nw = (int64_t)t.nt * T::N + 32 * NI * wn, mw = t.m_beg + 32 * MI * wm;
    if constexpr (KW > 1) {
      // the KW partial sums in order: wave kw finishes values VPW kw .. of each block's 16
      constexpr int VPW = 16 / KW;
      float* const red = reinterpret_cast<float*>(free);
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        if (i) lds_barrier();  // the last 32 slots' have been read
#pragma unroll
        for (int k = 0; k < NI; ++k)
#pragma unroll
          for (int v = 0; v < 16; ++v) red[((k * 16 + v) * G_WAVES + wave) * 64 + lane] = acc[i][k][v];
        lds_barrier();
#pragma unroll
        for (int k = 0; k < NI; ++k) {
          float o[VPW];
#pragma unroll
          for (int v = 0; v < VPW; ++v) {
            const int at = ((k * 16 + VPW * kw + v) * G_WAVES + part) * 64 + lane;
            o[v] = red[at];
#pragma unroll
            for (int w = 1; w < KW; ++w) o[v] += red[at + w * T::SHARE * 64];
          }
          if (32 * i + l32 < mine) {
#pragma unroll
            for (int v = 0; v < VPW; v += 2) {
              const int b = VPW * kw + v;
              const int64_t n = nw + 32 * k + 8 * (b >> 2) + 4 * half + (b & 3);
              uint16_t* const to = g.out + (mw + 32 * i + l32) * g.N + n;
              const uint32_t two = pack2<DT>(o[v], o[v + 1]);
              if (n + 1 < g.N && ((uintptr_t)to & 3) == 0) {
                *reinterpret_cast<uint32_t*>(to) = two;
              } else {
                if (n < g.N) to[0] = (uint16_t)two;
                if (n + 1 < g.N) to[1] = (uint16_t)(two >> 16);
              }
            }
          }
        }
      }
    } else if constexpr (!ACT) {
      // 32 slots at a time through the wave's part, for whole lines to memory
      uint8_t* const so = free + wave * (32 * T::OUT_ROW);
      constexpr int CH = T::OUT_ROW / 16;  // 16-byte chunks of a row
      const bool wide = g.N % 8 == 0 && ((uintptr_t)g.out & 15) == 0;
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int k = 0; k < NI; ++k)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *reinterpret_cast<uint2*>(so + l32 * T::OUT_ROW + 16 * ((4 * k + q) ^ (l32 & (CH - 1))) + 8 * half) =
                uint2{pack2<DT>(acc[i][k][4 * q], acc[i][k][4 * q + 1]), pack2<DT>(acc[i][k][4 * q + 2], acc[i][k][4 * q + 3])};
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int it = 0; it < 32 * CH / 64; ++it) {
          const int r = it * (64 / CH) + lane / CH, c = lane % CH;
          const u32x4 v = *reinterpret_cast<const u32x4*>(so + r * T::OUT_ROW + 16 * (c ^ (r & (CH - 1))));
          const int64_t n = nw + 8 * c;
          if (32 * i + r >= mine || n >= g.N) continue;
          uint16_t* const to = g.out + (mw + 32 * i + r) * g.N + n;
          if (wide) {
            *reinterpret_cast<u32x4*>(to) = v;
          } else {
#pragma unroll
            for (int b = 0; b < 8; ++b)
              if (n + b < g.N) to[b] = (uint16_t)(v[b >> 1] >> (16 * (b & 1)));
          }
        }
      }
    } else {
      // the gated activation over the gate's accumulators; a slot's 128 columns are 16 in each of two lanes of
      // each of the four waves that share the slots
      float* const s_max = reinterpret_cast<float*>(free);  // [M, 4]
      uint8_t* const s_q = free + T::M * 16;                // [M, 128], 16-byte chunks swizzled by the row
      const int64_t I = g.N / 2;
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        __builtin_amdgcn_sched_barrier(0);  // one block of 32 slots at a time: fewer registers
        float top = 0.f;
#pragma unroll
        for (int v = 0; v < 16; v += 2) {
          const f32x2 gate = unpack2<DT>(pack2<DT>(acc[i][0][v], acc[i][0][v + 1]));
          const f32x2 up = unpack2<DT>(pack2<DT>(acc[i][1][v], acc[i][1][v + 1]));
          const f32x2 sg = unpack2<DT>(pack2<DT>(silu_fast(gate.x), silu_fast(gate.y)));
          const f32x2 a = unpack2<DT>(pack2<DT>(sg.x * up.x, sg.y * up.y));
          acc[i][0][v] = a.x;
          acc[i][0][v + 1] = a.y;
          top = fmaxf(top, fmaxf(finite_abs(a.x), finite_abs(a.y)));
        }
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        if (half == 0) s_max[4 * (32 * (MI * wm + i) + l32) + wn] = top;
      }
      lds_barrier();
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        __builtin_amdgcn_sched_barrier(0);
        const int r = 32 * (MI * wm + i) + l32;
        const f32x4 m = *reinterpret_cast<const f32x4*>(s_max + 4 * r);
        const int e = e8m0_of(fmaxf(fmaxf(m.x, m.y), fmaxf(m.z, m.w)));
        const float inv = inv_scale(e);
        if (wn == 0 && half == 0 && 32 * i + l32 < mine) g.qs[(mw + 32 * i + l32) * g.q_sp + t.nt] = (uint8_t)e;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float a[4] = {acc[i][0][4 * q], acc[i][0][4 * q + 1], acc[i][0][4 * q + 2], acc[i][0][4 * q + 3]};
          *reinterpret_cast<uint32_t*>(s_q + r * 128 + 16 * ((2 * wn + (q >> 1)) ^ (r & 7)) + 8 * (q & 1) + 4 * half) =
              to_codes(a, inv);
        }
      }
      lds_barrier();
      for (int c = tid; c < T::M * 8; c += G_THREADS) {
        const int r = c >> 3;
        if (r < t.valid)
          *reinterpret_cast<u32x4*>(g.q + (t.m_beg + r) * I + (int64_t)t.nt * 128 + 16 * (c & 7)) =
              *reinterpret_cast<const u32x4*>(s_q + r * 128 + 16 * ((c & 7) ^ (r & 7)));
      }
    }
  }
  wait_vmcnt<0>();  // no DMA lands in LDS that is someone else's by then
}

bool raise_fp8_lds(const void* kernel, size_t bytes) {
  (void)hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  (void)hipGetLastError();
  return true;
}
template <int MW, int NW, int MI, int NI, int DT, bool WIDE, bool ACT>
void prepare_one() {
  static const bool done = raise_fp8_lds(reinterpret_cast<const void*>(&fp8_gemm_kernel<MW, NW, MI, NI, DT, WIDE, ACT>),
                                         Tile<MW, NW, MI, NI>::LDS);
  (void)done;
}

template <int MW, int NW, int MI, int NI, int DT, bool WIDE, bool ACT = false>
int launch_dt(const Fp8Args& g, unsigned blocks, hipStream_t st) {
  prepare_one<MW, NW, MI, NI, DT, WIDE, ACT>();
  fp8_gemm_kernel<MW, NW, MI, NI, DT, WIDE, ACT><<<blocks, G_THREADS, Tile<MW, NW, MI, NI>::LDS, st>>>(g);
  return check_launch("fp8_gemm");
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Each shape of tile: launch, one-time set-up, and what a call would take with it.
template <int MW, int NW, int MI, int NI>
struct Shape {
  typedef Tile<MW, NW, MI, NI> T;
  static int64_t tiles_at_most(const Fp8Args& g) {
    return (g.offsets ? (g.M < g.E ? g.M : g.E) + g.M / T::M : ceil_div(g.M, T::M)) * ceil_div(g.N, T::N);
  }
  static int launch(Fp8Args g, int dt, bool wide, hipStream_t st) {
    const int64_t tiles = tiles_at_most(g), cus = device_cu_count();
    if (tiles >= (int64_t)1 << 31) return set_error(USAF_ERR_INVALID, "fp8_gemm: too many tiles");
    g.n_nt = (int)ceil_div(g.N, T::N);
    const unsigned blocks = (unsigned)(ceil_div(tiles < cus ? tiles : cus, G_XCDS) * G_XCDS);
    if constexpr (NI == 2) {
      if (g.q)  // gate and up
        return dt == USAF_BF16 ? launch_dt<MW, NW, MI, NI, USAF_BF16, true, true>(g, blocks, st)
                               : launch_dt<MW, NW, MI, NI, USAF_F16, true, true>(g, blocks, st);
    }
    if (dt == USAF_BF16)
      return wide ? launch_dt<MW, NW, MI, NI, USAF_BF16, true>(g, blocks, st)
                  : launch_dt<MW, NW, MI, NI, USAF_BF16, false>(g, blocks, st);
    return wide ? launch_dt<MW, NW, MI, NI, USAF_F16, true>(g, blocks, st)
                : launch_dt<MW, NW, MI, NI, USAF_F16, false>(g, blocks, st);
  }
  static void prepare() {
    prepare_one<MW, NW, MI, NI, USAF_BF16, false, false>();
    prepare_one<MW, NW, MI, NI, USAF_BF16, true, false>();
    prepare_one<MW, NW, MI, NI, USAF_F16, false, false>();
    prepare_one<MW, NW, MI, NI, USAF_F16, true, false>();
    if constexpr (NI == 2) {
      prepare_one<MW, NW, MI, NI, USAF_BF16, true, true>();
      prepare_one<MW, NW, MI, NI, USAF_F16, true, true>();
    }
  }
  // Cycles of a CU, roughly: a step is bound by its matrix instructions or by its lines (24 bytes a cycle), a
  // tile has its ends, and the last round of tiles counts whole.  The shape of the least is taken.  Measured (us;
  // 256 x 256, 128 x 256, 128 x 128, 64 x 128, 64 x 64, 32 x 128, 32 x 64, 32 x 32; * the rule's, which is the fastest or
  // within 5 % of it but for 16 slots an expert, 6 %):
  //   rows x columns x contraction   8,192 x 14,336 x 4,096   438*  525  893  888  1,132 1,212 1,506 2,435
  //                                  4,096 x 4,096 x 2,048    35*   42   81   78   108   117   147   204
  //                                  1,024 x 4,096 x 2,048    27    20   21*  21   30    31    39    55
  //                                  333 x 1,411 x 2,027      35    23   23   13   9.7   9.8   7.8*  9.3
  //                                  33 x 4,096 x 2,048       19    18   18   11   8.7   9.1   7.0   6.0*
  //   128 experts' 768 x 2,048 gate and up (wide), 256 slots each  273  267* 308  373  444  441  531  700
  //                                                16 slots each   108  82*  99   81   99   77   93   111
  //   and their down projections, 256 slots each                   98*  104  153  163  257  252  387  587
  static double cycles(const Fp8Args& g, bool wide) {
    const double steps = (double)ceil_div(g.Kp / 128, T::KW);
    const double mfma = 2.0 * MI * NI * 2 * (wide ? 128 : 64), lines = (double)T::KW * (T::M + T::N) * 128 / 24;
    const double step = (mfma > lines ? mfma : lines) + 250, tile = steps * step + 1500;
    // slots of an expert: full tiles and on average half a tile
    const double m = g.offsets ? (double)(g.M < g.E ? g.M : g.E) * 0.5 + (double)g.M / T::M : (double)ceil_div(g.M, T::M);
    const double rounds = m * (double)ceil_div(g.N, T::N) / device_cu_count();
    return tile * (rounds < 1 ? 1 : g.offsets ? rounds + 0.5 : (double)(int64_t)(rounds + 0.999));
  }
};
typedef Shape<2, 4, 4, 2> S256x256;
typedef Shape<2, 4, 2, 2> S128x256;
typedef Shape<2, 4, 2, 1> S128x128;
typedef Shape<2, 4, 1, 1> S64x128;
typedef Shape<2, 2, 1, 1> S64x64;
typedef Shape<1, 4, 1, 1> S32x128;
typedef Shape<1, 2, 1, 1> S32x64;
typedef Shape<1, 1, 1, 1> S32x32;

typedef int (*Launch)(Fp8Args, int, bool, hipStream_t);
Launch best_shape(const Fp8Args& g, bool wide) {
  Launch best = S256x256::launch;
  double least = S256x256::cycles(g, wide);
  auto consider = [&](Launch f, double c) {
    if (c < least) {
      least = c;
      best = f;
    }
  };
  consider(S128x256::launch, S128x256::cycles(g, wide));
  consider(S128x128::launch, S128x128::cycles(g, wide));
  consider(S64x128::launch, S64x128::cycles(g, wide));
  consider(S64x64::launch, S64x64::cycles(g, wide));
  consider(S32x128::launch, S32x128::cycles(g, wide));
  consider(S32x64::launch, S32x64::cycles(g, wide));
  consider(S32x32::launch, S32x32::cycles(g, wide));
  return best;
}

}  // namespace

void prepare_fp8_kernels() {
  S256x256::prepare();
  S128x256::prepare();
  S128x128::prepare();
  S64x128::prepare();
  S64x64::prepare();
  S32x128::prepare();
  S32x64::prepare();
  S32x32::prepare();
}

}  // namespace usaf

using namespace usaf;

// Checks of a product's operands, and its arguments.
static int gemm_args(const char* what, const uint8_t* a, const uint8_t* a_scale, int64_t a_total, const int32_t* a_rows,
                     int64_t M, const uint8_t* w, const uint8_t* w_scale, const int32_t* offsets, int64_t E, int64_t N,
                     int64_t K, Fp8Args* args) {
  if (K == 0) return set_error(USAF_ERR_INVALID, "%s: need K >= 1", what);
  if (!a || !a_scale || !w || !w_scale) return set_error(USAF_ERR_INVALID, "%s: null pointer", what);
  if (!offsets && E != 1) return set_error(USAF_ERR_INVALID, "%s: more than one expert needs offsets", what);
  if (!a_rows && M > a_total) return set_error(USAF_ERR_INVALID, "%s: more slots than rows", what);
  if (E > Q_MAX_E) return set_error(USAF_ERR_UNSUPPORTED, "%s: at most %d experts", what, Q_MAX_E);
  if (((uintptr_t)a | (uintptr_t)w) % 16 || (uintptr_t)a_scale % 4)
    return set_error(USAF_ERR_INVALID, "%s: codes must be 16-byte and scales 4-byte aligned", what);
  Fp8Args& g = *args;
  g = Fp8Args{};
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
  // 32-bit offsets: gathered rows, a tile of 256 rows of either operand, the weight's scales
  if ((a_rows && a_total * g.Kp >= (int64_t)1 << 32) || 256 * g.Kp >= (int64_t)1 << 32 ||
      E * ((N + 127) / 128) * (g.Kp / 128) >= (int64_t)1 << 31)
    return set_error(USAF_ERR_UNSUPPORTED, "%s: operands past 4 GiB of gathered rows or 2 GiB of scales", what);
  return USAF_OK;
}

static int gemm_sizes(const char* what, int64_t a_total, int64_t M, int64_t E, int64_t N, int64_t K, int32_t dtype) {
  if (M < 0 || N < 0 || K < 0 || E < 1 || N > 1 << 24 || K > 1 << 24 || M > 0x7FFFFFFF || a_total < 0)
    return set_error(USAF_ERR_INVALID, "%s: bad size M=%lld N=%lld K=%lld E=%lld", what, (long long)M, (long long)N,
                     (long long)K, (long long)E);
  if (dtype != USAF_BF16 && dtype != USAF_F16) return set_error(USAF_ERR_INVALID, "%s: dtype must be fp16 or bf16", what);
  return USAF_OK;
}

extern "C" int usaf_hip_fp8_gemm(const uint8_t* a, const uint8_t* a_scale, int64_t a_total, const int32_t* a_rows, int64_t M,
                                 const uint8_t* w, const uint8_t* w_scale, const int32_t* offsets, int64_t E, int64_t N,
                                 int64_t K, int32_t dtype, int32_t wide, void* out, void* stream) {
  if (int rc = gemm_sizes("fp8_gemm", a_total, M, E, N, K, dtype)) return rc;
  if (M == 0 || N == 0) return clear_error();
  Fp8Args g;
  if (int rc = gemm_args("fp8_gemm", a, a_scale, a_total, a_rows, M, w, w_scale, offsets, E, N, K, &g)) return rc;
  if (!out || (uintptr_t)out % 2) return set_error(USAF_ERR_INVALID, "fp8_gemm: null or misaligned output");
  g.out = reinterpret_cast<uint16_t*>(out);
  return best_shape(g, wide != 0)(g, dtype, wide != 0, as_stream(stream));
}

// Whether the gate-and-up product may end in the gated activation's codes: on the tiles of 256
// columns, which the rule on sizes takes for all but the smallest calls, while an expert's gate rows
// stay within the 32-bit offsets.
static bool gate_up_ok(const Fp8Args& g) {
  const Launch best = best_shape(g, true);
  return (best == S256x256::launch || best == S128x256::launch) && (g.N / 2 + 128) * g.Kp < (int64_t)1 << 32;
}

extern "C" int usaf_hip_fp8_gate_up_ok(int64_t M, int64_t E, int64_t I, int64_t K) {
  if (M < 1 || E < 1 || E > Q_MAX_E || I < 1 || K < 1 || I % FP8_BLOCK || I > 1 << 23 || K > 1 << 24 || M > 0x7FFFFFFF) return 0;
  Fp8Args g{};
  static const int32_t grouped = 0;
  g.offsets = &grouped;  // not read
  g.Kp = (K + FP8_BLOCK - 1) / FP8_BLOCK * FP8_BLOCK;
  g.N = 2 * I;
  g.E = (int)E;
  g.M = M;
  return gate_up_ok(g) ? 1 : 0;
}

extern "C" int usaf_hip_fp8_gate_up(const uint8_t* a, const uint8_t* a_scale, int64_t a_total, const int32_t* a_rows,
                                    int64_t M, const uint8_t* w, const uint8_t* w_scale, const int32_t* offsets, int64_t E,
                                    int64_t I, int64_t K, int32_t dtype, uint8_t* q, uint8_t* s, void* stream) {
  if (I < 0 || I % FP8_BLOCK || I > 1 << 23)
    return set_error(USAF_ERR_INVALID, "fp8_gate_up: I must be a multiple of %d, got %lld", FP8_BLOCK, (long long)I);
  if (int rc = gemm_sizes("fp8_gate_up", a_total, M, E, 2 * I, K, dtype)) return rc;
  if (M == 0 || I == 0) return clear_error();
  Fp8Args g;
  if (int rc = gemm_args("fp8_gate_up", a, a_scale, a_total, a_rows, M, w, w_scale, offsets, E, 2 * I, K, &g)) return rc;
  if (!offsets || !q || !s || (uintptr_t)q % 16)
    return set_error(USAF_ERR_INVALID, "fp8_gate_up: null pointer, or codes not 16-byte aligned");
  if (!gate_up_ok(g)) return set_error(USAF_ERR_UNSUPPORTED, "fp8_gate_up: not at this size (usaf_hip_fp8_gate_up_ok)");
  g.q = q;
  g.qs = s;
  g.q_sp = (int)usaf_hip_fp8_scale_stride(I);
  return best_shape(g, true)(g, dtype, true, as_stream(stream));
}

extern "C" int64_t usaf_hip_fp8_linear_ws_bytes(int64_t M, int64_t K) {
  if (M < 0 || K < 0 || K > 1 << 24 || M > 0x7FFFFFFF) return -1;
  return fp8_small_ok(M, K) ? 0 : M * ((K + FP8_BLOCK - 1) / FP8_BLOCK * FP8_BLOCK + usaf_hip_fp8_scale_stride(K));
}

extern "C" int usaf_hip_fp8_linear(const void* x, int32_t dtype, int64_t M, int64_t K, int64_t ld, const uint8_t* w,
                                   const uint8_t* w_scale, int64_t N, void* out, void* ws, int64_t ws_bytes, void* stream) {
  const int64_t need = usaf_hip_fp8_linear_ws_bytes(M, K);
  if (need < 0) return set_error(USAF_ERR_INVALID, "fp8_linear: bad size M=%lld K=%lld", (long long)M, (long long)K);
  if (M == 0 || N == 0) return clear_error();
  if (N < 0 || N > 1 << 24 || ld < K || K == 0)
    return set_error(USAF_ERR_INVALID, "fp8_linear: need 0 <= N <= 2^24 and ld >= K >= 1");
  if (dtype != USAF_BF16 && dtype != USAF_F16) return set_error(USAF_ERR_INVALID, "fp8_linear: dtype must be fp16 or bf16");
  if (!x || !w || !w_scale || !out) return set_error(USAF_ERR_INVALID, "fp8_linear: null pointer");
  if ((uintptr_t)w % 16 || ((uintptr_t)out | (uintptr_t)x) % 2)
    return set_error(USAF_ERR_INVALID, "fp8_linear: codes must be 16-byte, rows and output 2-byte aligned");
  if (fp8_small_ok(M, K)) return fp8_small(x, dtype, M, K, ld, w, w_scale, N, out, as_stream(stream));
  if (!ws || ws_bytes < need)
    return set_error(USAF_ERR_INVALID, "fp8_linear: workspace of %lld bytes, need %lld", (long long)ws_bytes, (long long)need);
  uint8_t* const q = reinterpret_cast<uint8_t*>(ws);
  uint8_t* const s = q + M * ((K + FP8_BLOCK - 1) / FP8_BLOCK * FP8_BLOCK);
  if (int rc = usaf_hip_fp8_quantize_rows(x, dtype, M, K, ld, nullptr, q, s, stream)) return rc;
  return usaf_hip_fp8_gemm(q, s, M, nullptr, M, w, w_scale, nullptr, 1, N, K, dtype, 0, out, stream);
}

// ---- an 8-bit expert layer between the bucketing and the weighted sums, in one call each way --------

extern "C" int64_t usaf_hip_fp8_experts_fwd_ws_bytes(int64_t S, int64_t I) {
  if (S < 0 || I < 0 || S > 0x7FFFFFFF || I > 1 << 23) return -1;
  return S * (I + usaf_hip_fp8_scale_stride(I));
}

extern "C" int usaf_hip_fp8_experts_fwd(const uint8_t* x, const uint8_t* x_scale, int64_t T, const int32_t* token_idx,
                                        const int32_t* offsets, int64_t S, int64_t E, int64_t H, int64_t I, int32_t dtype,
                                        const uint8_t* gate_up, const uint8_t* gate_up_scale, const uint8_t* down,
                                        const uint8_t* down_scale, void* gu, void* act, void* y, void* ws, int64_t ws_bytes,
                                        void* stream) {
  const int64_t need = usaf_hip_fp8_experts_fwd_ws_bytes(S, I);
  if (need < 0 || H < 1 || H % FP8_BLOCK || I < 1 || I % FP8_BLOCK)
    return set_error(USAF_ERR_INVALID, "fp8_experts_fwd: H and I must be positive multiples of %d", FP8_BLOCK);
  if (S == 0) return clear_error();
  if (!token_idx || !offsets || !y) return set_error(USAF_ERR_INVALID, "fp8_experts_fwd: null pointer");
  if (!ws || (uintptr_t)ws % 16 || ws_bytes < need)
    return set_error(USAF_ERR_INVALID, "fp8_experts_fwd: a workspace of %lld bytes, 16-byte aligned", (long long)need);
  uint8_t *const q = reinterpret_cast<uint8_t*>(ws), *const s = q + S * I;
  if (!gu && !act) {
    if (int rc = usaf_hip_fp8_gate_up(x, x_scale, T, token_idx, S, gate_up, gate_up_scale, offsets, E, I, H, dtype, q, s, stream))
      return rc;
  } else {
    if (int rc = usaf_hip_fp8_gemm(x, x_scale, T, token_idx, S, gate_up, gate_up_scale, offsets, E, 2 * I, H, dtype, 1, gu,
                                   stream))
      return rc;
    if (int rc = usaf_hip_fp8_swiglu(gu, S, I, dtype, offsets + E, act, q, s, stream)) return rc;
  }
  return usaf_hip_fp8_gemm(q, s, S, nullptr, S, down, down_scale, offsets, E, H, I, dtype, 0, y, stream);
}

// The quantized gradients of y and of gu, one behind the other in the same place, then d(act).
static int64_t bwd_rows_bytes(int64_t S, int64_t H, int64_t I) {
  const int64_t a = S * (H + usaf_hip_fp8_scale_stride(H)), b = S * (2 * I + usaf_hip_fp8_scale_stride(2 * I));
  return ((a > b ? a : b) + 255) / 256 * 256;  // d(act) starts a cache line
}

extern "C" int64_t usaf_hip_fp8_experts_bwd_ws_bytes(int64_t S, int64_t H, int64_t I) {
  if (S < 0 || H < 0 || I < 0 || S > 0x7FFFFFFF || H > 1 << 24 || I > 1 << 23) return -1;
  return bwd_rows_bytes(S, H, I) + 2 * S * I;
}

extern "C" int usaf_hip_fp8_experts_bwd(const void* dout, const void* y, const void* gu, const int32_t* token_idx,
                                        const float* slot_w, const int32_t* offsets, int64_t S, int64_t E, int64_t H, int64_t I,
                                        int32_t dtype, const uint8_t* down_t, const uint8_t* down_t_scale,
                                        const uint8_t* gate_up_t, const uint8_t* gate_up_t_scale, void* dcur, void* dgu,
                                        void* dx_slots, void* dweights, void* ws, int64_t ws_bytes, void* stream) {
  const int64_t need = usaf_hip_fp8_experts_bwd_ws_bytes(S, H, I);
  if (need < 0 || H < 1 || H % FP8_BLOCK || I < 1 || I % FP8_BLOCK)
    return set_error(USAF_ERR_INVALID, "fp8_experts_bwd: H and I must be positive multiples of %d", FP8_BLOCK);
  if (S == 0) return clear_error();
  if (!gu || !dx_slots) return set_error(USAF_ERR_INVALID, "fp8_experts_bwd: null pointer");
  if (!ws || (uintptr_t)ws % 16 || ws_bytes < need)
    return set_error(USAF_ERR_INVALID, "fp8_experts_bwd: a workspace of %lld bytes, 16-byte aligned", (long long)need);
  uint8_t* const q = reinterpret_cast<uint8_t*>(ws);
  void* const dact = q + bwd_rows_bytes(S, H, I);
  if (int rc = usaf_hip_fp8_combine_bwd(dout, y, token_idx, slot_w, offsets, S, E, H, dtype, dcur, q, q + S * H, dweights, stream))
    return rc;
  if (int rc = usaf_hip_fp8_gemm(q, q + S * H, S, nullptr, S, down_t, down_t_scale, offsets, E, I, H, dtype, 1, dact, stream))
    return rc;
  if (int rc = usaf_hip_fp8_swiglu_bwd(gu, dact, S, I, dtype, offsets + E, dgu, q, q + 2 * S * I, stream)) return rc;
  return usaf_hip_fp8_gemm(q, q + 2 * S * I, S, nullptr, S, gate_up_t, gate_up_t_scale, offsets, E, H, 2 * I, dtype, 0, dx_slots,
                           stream);
}

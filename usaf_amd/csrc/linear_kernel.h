// The product with one weight, 16-bit or 4-bit, as linear_dense.hip and linear_q4.hip build it:
//
//   C[m, n] = sum_k A[m, k] W[n, k];   out = dt(C),  or with G = C's gate half and U its up half
//   out = dt(silu(G) U), and for a backward dt(G), dt(U) or their 8-bit blocks Q(G), Q(U)
//
// The weights are the matrix instruction's A operand, the rows of A ("slots") its B operand, so a lane's
// accumulator holds 4 consecutive columns of one slot.  Gated tiles take 16 rows of the gate and the same 16 of up into
// each 32 x 32 block: values v and v + 8 of a lane are then a column's gate and up.
//
// A block of eight or four waves has tiles of 32 MW MI slots x 32 NW NI weight rows; KW of its waves split the
// contraction's blocks of 64.  Blocks stay (one a CU) and walk a die's run of the tile list.  Both operands come by LDS
// DMA, 128-byte lines, into a ring of NS stages, straight across tile ends.  16-byte chunks are XOR-swizzled by the row
// (by the DMA's source address), which spreads the fragment reads over the banks.  A step has four slices, 16 of the
// contraction for each half of the lanes; a slice's fragments are read while the one before it is multiplied, the first
// of the next step's behind the step's one barrier, in front of its last slice: there the next stage has landed and this
// one has been read, so its next lines are sent for.
//
// 4-bit weights (MW = 1: a weight row's codes belong to one wave) are dequantized as they come out of LDS, into the
// matrix instruction's operand registers: dt(fp16(fp16(q s) + z)), the codec's value bit for bit.
//
// What bounds it (bf16).  Large tiles: the matrix instructions and the clock that they leave; 1.27 us of a 256 x 256 x 64 step's
// 1.6 are theirs alone.  8,192 x 14,336 x 4,096 takes 720 to 770 us (1.25 to 1.34 PFLOP/s); the library's product 606, under the
// same clock.  Smaller tiles: the trip of their lines, so stages count: 2,048 x 2,048 of 16,384 took 182 us with two stages of 128 x 256
// tiles and takes 136 to 150 with three.  4-bit weights: the dequantization's vector instructions, 1.20 us a step of 128 x 256 x 64 against 0.90.
#pragma once

#include "dma.h"
#include "fp8.h"
#include "linear.h"

#include <type_traits>

namespace usaf {
namespace {

constexpr int L_XCDS = 8;  // accelerator dies, blocks dispatched round-robin over them

enum { LIN_STORE = 0, LIN_GATED = 1, LIN_CK8 = 2 };

template <int WAVES, int MW, int NW, int MI, int NI, bool Q4, int EPI>
struct LinTile {
  static constexpr int KW = WAVES / (MW * NW), NB = NW * NI;
  static constexpr int M = 32 * MW * MI, N = 32 * NB;
  static constexpr int COLS = EPI == LIN_STORE ? N : N / 2;          // columns of out
  static constexpr int W_ROW = Q4 ? 32 : 128;                        // bytes of a weight row's 64 values
  static constexpr int A_BYTES = M * 128, W_BYTES = N * W_ROW;
  static constexpr int S_WORDS = Q4 ? (N + 63) / 64 : 0;             // instructions of 64 scale words
  static constexpr int SLAB = A_BYTES + W_BYTES + 256 * S_WORDS, STAGE = KW * SLAB;
  // the results' way out: partial sums of KW waves, then 32 EW slots' rows of out and of what is kept
  static constexpr int RED = KW > 1 ? WAVES * NI * 16 * 64 * 4 : 0;
  static constexpr int OUT_ROW = 2 * COLS, KEPT_ROW = EPI == LIN_GATED ? 2 * N : EPI == LIN_CK8 ? N : 0;
  static constexpr int SLOT_ENDS = OUT_ROW + KEPT_ROW;
  // (of one wave row's slots where that leaves room for one more stage)
  static constexpr int stages(int ew) { return (160 * 1024 - RED - 32 * ew * SLOT_ENDS) / STAGE; }
  static constexpr int EW = KW > 1 || EPI == LIN_CK8 || stages(MW) == stages(1) || stages(MW) >= 4 ? MW : 1, ER = 32 * EW;
  static constexpr int ENDS = RED + ER * SLOT_ENDS;
  static constexpr int NS = stages(EW) > 4 ? 4 : stages(EW);
  static constexpr int LDS = NS * STAGE + ENDS;
  // DMA instructions of a wave and step: the rows of its own k-block, shared by the MW NW waves that have it
  static constexpr int SHARE = MW * NW;
  static constexpr int W_RPI = 1024 / W_ROW;                         // weight rows of an instruction
  static constexpr int A_DMA = (M / 8 + SHARE - 1) / SHARE, W_DMA = (N / W_RPI + SHARE - 1) / SHARE;
  static constexpr int S_DMA = Q4 ? (S_WORDS + SHARE - 1) / SHARE : 0, DMAS = A_DMA + W_DMA + S_DMA;
  static_assert(NS >= 2 && MW * NW * KW == WAVES && (!Q4 || MW == 1), "tile");
  static_assert(EPI != LIN_CK8 || (N == 256 && KW == 1 && EW == MW), "a tile has whole blocks of 128 columns");
};

// Four columns' values of 16 of four rows: each 16 lanes' 16 addresses are of 8 bytes, lane 4 r + c's of row r, and lane i
// gets column i of the four rows.
typedef short s16x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ uint2 read_turned(const uint8_t* p) {
  typedef __attribute__((address_space(3))) s16x4* Ptr;
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Ptr)p));
}

template <int WAVES, int MW, int NW, int MI, int NI, int DT, bool Q4, int EPI, int TR>
__global__ __launch_bounds__(64 * WAVES, WAVES / 4) void linear_kernel(const LinArgs g) {
  typedef LinTile<WAVES, MW, NW, MI, NI, Q4, EPI> T;
  constexpr int THREADS = 64 * WAVES;
  constexpr int KW = T::KW, NB = T::NB;
  constexpr bool TW = TR >= 1, TA = TR == 2;  // stored with the contraction's index first
  constexpr int W_CH = T::N / 8, A_CH = T::M / 8;  // chunks of such a row
  static_assert(!TW || (!Q4 && EPI == LIN_STORE && KW == 1 && W_CH % 16 == 0 && W_CH <= 32), "tile");
  static_assert(!TA || (A_CH % 16 == 0 && A_CH <= 32), "tile");
  constexpr bool GATED = EPI != LIN_STORE, PARTS = !GATED && WAVES == 8;  // PARTS: takes a contraction in parts
  extern __shared__ __attribute__((aligned(16))) uint8_t sm[];
  const uint32_t sm_lds = (uint32_t)(uintptr_t)(lds_void_ptr)sm;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, half = lane >> 5;
  const int kw = wave / T::SHARE, part = wave % T::SHARE, wm = part % MW, wn = part / MW;

  // ---- the block's tiles: its die's run of the list, every blocks-of-a-die-th; what a die's blocks share at a
  //      time, eight slot tiles of one weight tile, sits in its L2
  const int m_tiles = (int)((g.M + T::M - 1) / T::M);
  const int tiles = m_tiles * g.n_nt, units = tiles * g.parts;  // a part of the contraction after the other
  const int per = (units + L_XCDS - 1) / L_XCDS, stride = (int)gridDim.x / L_XCDS, xcd = (int)blockIdx.x % L_XCDS;
  const int run = xcd * per, end = run + per < units ? run + per : units, id0 = run + (int)blockIdx.x / L_XCDS;
  if (id0 >= end) return;  // block-uniform
  struct Place {
    int valid, nt, part, s_beg, s_end;
    int64_t m_beg;
  };
  const int nkb = (int)(g.K / 64), all_steps = (nkb + KW - 1) / KW;
  const int64_t s_row = 4 * (GATED ? 2 * g.N : g.N);  // bytes of a group's words
  auto place = [&](int unit) {
    constexpr int GROUP = 8;
    Place t;
    t.part = g.parts > 1 ? unit / tiles : 0;
    t.s_beg = all_steps * t.part / g.parts;
    t.s_end = all_steps * (t.part + 1) / g.parts;
    const int id = unit - t.part * tiles;
    const int band = id / (GROUP * g.n_nt), rest = id - band * GROUP * g.n_nt;
    const int tall = m_tiles - band * GROUP < GROUP ? m_tiles - band * GROUP : GROUP;
    t.nt = rest / tall;
    t.m_beg = (int64_t)(band * GROUP + rest - t.nt * tall) * T::M;
    t.valid = g.M - t.m_beg < T::M ? (int)(g.M - t.m_beg) : T::M;
    return t;
  };
  const int64_t up_rows = GATED ? g.N : 0;

  // ---- the DMA stream: uniform bases, 32-bit lane offsets.  Instruction i of wave `part` fills rows
  //      (SHARE i + part) of 8 (4-bit: 32) of the k-block; lane l of 128-byte rows chunk l % 8 of row l / 8.  A tile row r is
  //      column r of out's tile, gated: 16 (r / 32) + r % 16, of the gate for r / 16 even
  int i_id = id0, i_step = 0, i_end = 0, i_stage = 0;
  const uint8_t *a_base, *w_base, *s_base = nullptr;
  uint32_t a_off[T::A_DMA], w_off[T::W_DMA], s_off[T::S_DMA > 0 ? T::S_DMA : 1];
  auto open = [&]() {
    const Place t = place(i_id);
    const int64_t n0 = (int64_t)t.nt * T::COLS;
    i_step = t.s_beg;
    i_end = t.s_end;
    auto column = [&](int r) {  // from n0, of a column that exists
      const int c = GATED ? 16 * (r >> 5) + (r & 15) : r;
      return n0 + c < g.N ? (int64_t)c : g.N - 1 - n0;
    };
    a_base = uniform(g.A + t.m_beg * (TA ? 2 : g.lda));
    w_base = uniform(g.W + n0 * (TW ? 2 : g.ldw));
    // chunk p of row r holds the row's chunk p ^ 4 (r % 4); columns past the last: its chunk again
    auto chunk = [&](int at, int ch, int have, int64_t ld) {
      const int r = 64 / ch * at + lane / ch, c = (lane % ch) ^ (4 * (r & 3));
      return (uint32_t)(r * ld) + 16 * (c < have ? c : have - 1);
    };
#pragma unroll
    for (int i = 0; i < T::A_DMA; ++i) {
      const int r = (8 * (T::SHARE * i + part) + (lane >> 3)) % T::M;  // (of few rows, some twice)
      if constexpr (TA) a_off[i] = chunk((T::SHARE * i + part) % A_CH, A_CH, t.valid / 8, g.lda);
      else a_off[i] = (uint32_t)((r < t.valid ? r : t.valid - 1) * g.lda) + 16 * ((lane & 7) ^ g_swz(r));
    }
#pragma unroll
    for (int i = 0; i < T::W_DMA; ++i) {
      if constexpr (TW) {
        const int64_t left = g.N - n0;
        w_off[i] = chunk((T::SHARE * i + part) % W_CH, W_CH, left < T::N ? (int)left / 8 : W_CH, g.ldw);
      } else if constexpr (Q4) {
        const int r = (32 * (T::SHARE * i + part) + (lane >> 1)) % T::N;
        const int64_t n = column(r) + (GATED && (r & 16) ? up_rows : 0);
        w_off[i] = (uint32_t)(n * g.ldw) + 16 * ((lane & 1) ^ (r >> 3 & 1));
      } else {
        const int r = (8 * (T::SHARE * i + part) + (lane >> 3)) % T::N;
        w_off[i] = (uint32_t)(column(r) * g.ldw) + 16 * ((lane & 7) ^ g_swz(r));
      }
    }
    if constexpr (Q4) {
      s_base = uniform(reinterpret_cast<const uint8_t*>(g.sz + n0));
#pragma unroll
      for (int i = 0; i < T::S_DMA; ++i) {
        const int r = (64 * (T::SHARE * i + part) + lane) % T::N;
        s_off[i] = (uint32_t)((column(r) + (GATED && (r & 16) ? up_rows : 0)) * 4);
      }
    }
  };
  // One step's DMAs, in T::DMAS pieces: begin, the pieces, advance
  uint32_t i_to = 0;
  int i_k = 0;
  const uint8_t *i_a = nullptr, *i_w = nullptr;
  auto begin = [&]() {
    const int kb = i_step * KW + kw;
    i_k = kb < nkb ? kb : nkb - 1;
    i_to = (uint32_t)__builtin_amdgcn_readfirstlane((int)(sm_lds + i_stage * T::STAGE + kw * T::SLAB));
    i_a = a_base + (int64_t)i_k * (TA ? 64 * g.lda : 128);
    i_w = w_base + (int64_t)i_k * (TW ? 64 * g.ldw : T::W_ROW);
  };
  // (readfirstlane of what is uniform already is a move at most; without it the compiler may hold it in vector registers)
  auto to_lds = [](uint32_t at) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)at); };
  auto from = [](const uint8_t* p) { return Q4 ? uniform(p) : p; };
  auto piece = [&](int p) {
    if (p < T::W_DMA) {
      const int at = T::SHARE * p + part;  // wave-uniform
      const uint8_t* base = i_w;
      if (!Q4 && GATED && (at & 2)) base += up_rows * g.ldw;
      g_dma16(from(base), w_off[p < T::W_DMA ? p : 0], to_lds(i_to + T::A_BYTES + at * 1024 % T::W_BYTES));
    } else if (p < T::W_DMA + T::A_DMA) {
      const int i = p - T::W_DMA;
      g_dma16(from(i_a), a_off[i < T::A_DMA ? i : 0], to_lds(i_to + (T::SHARE * i + part) * 1024 % T::A_BYTES));
    } else if (p < T::DMAS) {
      const int i = p - T::W_DMA - T::A_DMA, s = (T::SHARE * i + part) % (T::S_WORDS > 0 ? T::S_WORDS : 1);
      g_dma4(from(s_base + (i_k >> 1) * s_row), s_off[i < T::S_DMA ? i : 0], to_lds(i_to + T::A_BYTES + T::W_BYTES + 256 * s));
    }
  };
  auto advance = [&]() {
    i_stage = i_stage + 1 == T::NS ? 0 : i_stage + 1;
    if (++i_step == i_end) {
      if (i_id + stride < end) {
        i_id += stride;
        open();
      } else {
        i_step = i_end - 1;  // past the block's last step: that one again, which nobody reads
      }
    }
  };

  // ---- fragments.  Half h of a 32 x 32 x 16 product's 64 lanes has k = 32 h + 8 j + [0, 8) of a step's product j, on
  //      both sides.  A slice is product j's of all the wave's blocks; the next slice's come while one is multiplied
  u32x4 wf[2][NI], af[2][MI], codes[Q4 ? NI : 1];
  uint32_t scale[Q4 ? NI : 1];
  // fragment n of a slice's NI of the weights (4-bit: a step's codes, in front of its first slice) and MI of the slots
  auto load_one = [&](int stage, int j, int n, u32x4(&w)[NI], u32x4(&a)[MI]) {
    const uint8_t* const sa = sm + stage * T::STAGE + kw * T::SLAB;
    const uint8_t* const sw = sa + T::A_BYTES;
    auto word = [&](const uint8_t* rows, int r, int c) {
      return *reinterpret_cast<const u32x4*>(rows + r * 128 + 16 * (c ^ g_swz(r)));
    };
    // block b's values of rows 32 half + 8 j + [0, 8) of the contraction
    auto turned = [&](const uint8_t* rows, int ch, int b) {
      const int r = lane >> 2 & 3, c = 4 * b + 2 * (lane >> 4 & 1) + (lane >> 1 & 1);
      const uint8_t* const at = rows + (32 * half + 8 * j + r) * 16 * ch + 16 * (c ^ 4 * r) + 8 * (lane & 1);
      const uint2 lo = read_turned(at), hi = read_turned(at + 64 * ch);
      return u32x4{lo.x, lo.y, hi.x, hi.y};
    };
    if (n < NI) {
      const int k = n, r = 32 * (NI * wn + k) + l32;
      if constexpr (TW) {
        w[k] = turned(sw, W_CH, NI * wn + k);
      } else if constexpr (!Q4) {
        w[k] = word(sw, r, 4 * half + j);
      } else if (j == 0) {
        codes[k] = *reinterpret_cast<const u32x4*>(sw + r * 32 + 16 * (half ^ (r >> 3 & 1)));
        scale[k] = reinterpret_cast<const uint32_t*>(sw + T::W_BYTES)[r];
      }
    } else if (n < NI + MI) {
      if constexpr (TA) a[n - NI] = turned(sa, A_CH, MI * wm + n - NI);
      else a[n - NI] = word(sa, 32 * (MI * wm + n - NI) + l32, 4 * half + j);
    }
  };
  auto load_slice = [&](int stage, int j, u32x4(&w)[NI], u32x4(&a)[MI]) {
#pragma unroll
    for (int n = 0; n < NI + MI; ++n) load_one(stage, j, n, w, a);
  };
  // 4-bit: pair n of a slice's 4 NI
  auto dequant = [&](int j, int n, u32x4(&w)[NI]) {
    if constexpr (Q4) {
      const int k = n >> 2;
      const f16 s = __builtin_bit_cast(f16, (uint16_t)scale[k]), z = __builtin_bit_cast(f16, (uint16_t)(scale[k] >> 16));
      w[k][n & 3] = dq_pair<DT>(codes[k][j], n & 3, f16x2{s, s}, f16x2{z, z});
    }
  };

  f32x16 acc[MI][NI];
  int stage = 0;
  // A step's DMAs go out behind its barrier.  Of eight waves, a SIMD's two send at different times (one in front of the last
  // slice, one in front of the next step's first), so that one has products while the other waits for the address unit:
  // all at once cost 4 % of a large product.  Four waves send between the products of the same two slices.
  const bool early = wave < WAVES / 2;
  constexpr int HALF = (T::DMAS + 1) / 2;
  auto send = [&](int first, int last) {
#pragma unroll
    for (int p = 0; p < T::DMAS; ++p)
      if (p >= first && p < last) piece(p);
  };
  auto next_stage = [&]() {
    wait_vmcnt<(T::NS - 2) * T::DMAS>();  // the wave's DMAs of the next stage (and what is older) have landed
    lds_barrier();                        // and everyone's; this stage has been read
    stage = stage + 1 == T::NS ? 0 : stage + 1;
  };
  open();
  for (int s = 0; s < T::NS - 1; ++s) {
    begin();
    send(0, T::DMAS);
    advance();
  }
  stage = T::NS - 1;
  next_stage();
  load_slice(0, 0, wf[0], af[0]);
#pragma unroll
  for (int n = 0; n < 4 * NI; ++n) dequant(0, n, wf[0]);
  begin();
  if (WAVES == 4) send(0, HALF);
  else if (early) send(0, T::DMAS);
  for (int id = id0; id < end; id += stride) {
    const Place t = place(id);
    const int mine = t.valid - 32 * MI * wm;  // slots of the wave's part
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int k = 0; k < NI; ++k) acc[i][k] = f32x16{};
    for (int step = t.s_beg; step < t.s_end; ++step) {
      const bool mine_too = KW == 1 || step * KW + kw < nkb;  // wave-uniform
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        u32x4(&w)[NI] = wf[j & 1];
        u32x4(&x)[MI] = af[j & 1];
        if (j == 3) next_stage();
        if constexpr (WAVES == 8) {
          load_slice(stage, (j + 1) & 3, wf[(j + 1) & 1], af[(j + 1) & 1]);
          if (j == 3) begin();
          if (early ? j == 3 : j == 0) send(0, T::DMAS);
          __builtin_amdgcn_sched_barrier(0);
          // 4-bit: the next slice's weights are dequantized between this one's products, 4 / MI pairs behind each
          auto products = [&](auto with) {
#pragma unroll
            for (int i = 0; i < MI; ++i) {
#pragma unroll
              for (int k = 0; k < NI; ++k)
                if constexpr (decltype(with)::value) acc[i][k] = mfma32<DT>(w[k], x[i], acc[i][k]);
              if constexpr (Q4) {
                if (MI > 1) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int n = 4 * NI * i / MI; n < 4 * NI * (i + 1) / MI; ++n) dequant((j + 1) & 3, n, wf[(j + 1) & 1]);
                if (MI > 1) __builtin_amdgcn_sched_barrier(0);
              }
            }
          };
          if (mine_too) products(std::true_type());
          else products(std::false_type());
        } else {
          // one wave a SIMD: reads and DMAs in turn between the products
          static_assert(KW == 1 && 2 * (MI + NI) <= MI * NI && 2 * HALF <= MI * NI, "they fit between");
          if (j == 3) begin();
#pragma unroll
          for (int n = 0; n < MI * NI; ++n) {
            if (n % 2 == 0) load_one(stage, (j + 1) & 3, n / 2, wf[(j + 1) & 1], af[(j + 1) & 1]);
            else if (j == 3 && n / 2 < HALF) send(n / 2, n / 2 + 1);
            else if (j == 0 && HALF + n / 2 < T::DMAS) send(HALF + n / 2, HALF + n / 2 + 1);
            acc[n / NI][n % NI] = mfma32<DT>(w[n % NI], x[n / NI], acc[n / NI][n % NI]);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        if (j == 0) advance();
        __builtin_amdgcn_sched_barrier(0);
      }
    }

    // ---- results, the same 32 of EW of the wave rows' slots at a time through LDS, for whole lines to memory.  Wave kw
    //      finishes values VH kw + [0, VH) of a block's lower 16 rows and the same of its upper 16
    // (the lane's place is taken anew, or what hangs on it is computed ahead of the tiles and held in
    // registers that the steps lack)
    int tid_now = threadIdx.x;
    asm volatile("" : "+v"(tid_now));
    const int e_l32 = tid_now & 31, e_half = tid_now >> 5 & 1, e_lane = tid_now & 63;
    constexpr int VH = KW > 1 ? 8 / KW : 8, RL = VH < 4 ? VH : 4;
    uint8_t* const ends = sm + T::NS * T::STAGE;
    float* const red = reinterpret_cast<float*>(ends);
    uint8_t* const s_out = ends + T::RED;
    uint8_t* const s_kept = s_out + T::ER * T::OUT_ROW;
    const int64_t n0 = (int64_t)t.nt * T::COLS;
    // RL values to column c of row r of `row` bytes
    auto put = [&](uint8_t* rows, int row, int r, int c, const float* v) {
      uint8_t* const to = rows + r * row + 16 * ((c >> 3) ^ (r & (row / 16 - 1))) + 2 * (c & 7);
      if constexpr (RL == 4) *reinterpret_cast<uint2*>(to) = uint2{pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3])};
      else if constexpr (RL == 2) *reinterpret_cast<uint32_t*>(to) = pack2<DT>(v[0], v[1]);
      else *reinterpret_cast<uint16_t*>(to) = (uint16_t)pack2<DT>(v[0], v[0]);
    };
#pragma unroll
    for (int ih = 0; ih < MI * (MW / T::EW); ++ih) {
      const int i = ih / (MW / T::EW), h = ih % (MW / T::EW);
      if (32 * (MI * T::EW * h + i) >= t.valid) continue;  // block-uniform: no slots
      lds_barrier();  // the last slots' reads are done
      if (T::EW == MW || wm == h) {  // wave-uniform
      float lo[NI][VH], hi[NI][VH];
      if constexpr (KW > 1) {
#pragma unroll
        for (int k = 0; k < NI; ++k)
#pragma unroll
          for (int v = 0; v < 16; ++v) red[((k * 16 + v) * WAVES + wave) * 64 + e_lane] = acc[i][k][v];
        lds_barrier();
#pragma unroll
        for (int k = 0; k < NI; ++k)
#pragma unroll
          for (int v = 0; v < VH; ++v) {
            const int at = ((k * 16 + VH * kw + v) * WAVES + part) * 64 + e_lane;
            lo[k][v] = red[at];
            hi[k][v] = red[at + 8 * WAVES * 64];
#pragma unroll
            for (int w = 1; w < KW; ++w) {
              lo[k][v] += red[at + w * T::SHARE * 64];
              hi[k][v] += red[at + (8 * WAVES + w * T::SHARE) * 64];
            }
          }
      } else {
#pragma unroll
        for (int k = 0; k < NI; ++k)
#pragma unroll
          for (int v = 0; v < 8; ++v) {
            lo[k][v] = acc[i][k][v];
            hi[k][v] = acc[i][k][v + 8];
          }
      }
      if constexpr (PARTS) {
        if (g.parts > 1) {  // fp32 sums of a part of the contraction, RL columns at a time
          if (32 * i + e_l32 < mine) {
            float* const to = g.part + (t.part * g.M + t.m_beg + 32 * (MI * wm + i) + e_l32) * g.ldp;
#pragma unroll
            for (int k = 0; k < NI; ++k)
#pragma unroll
              for (int r0 = 0; r0 < VH; r0 += RL)
#pragma unroll
                for (int up = 0; up < 2; ++up) {
                  const int v = VH * (KW > 1 ? kw : 0) + r0;
                  const int64_t n = n0 + 32 * (NI * wn + k) + 16 * up + 8 * (v >> 2) + 4 * e_half + (v & 3);
                  const float* const f = up ? &hi[k][r0] : &lo[k][r0];
                  if (n < g.ldp) {
                    if constexpr (RL == 4) *reinterpret_cast<f32x4*>(to + n) = f32x4{f[0], f[1], f[2], f[3]};
                    else if constexpr (RL == 2) *reinterpret_cast<f32x2*>(to + n) = f32x2{f[0], f[1]};
                    else to[n] = f[0];
                  }
                }
          }
          continue;
        }
      }
      const int row = 32 * (wm % T::EW) + e_l32;
      if constexpr (EPI == LIN_CK8) {
        // a block's largest magnitude: the lane's columns, the other half's, the other waves'
        float* const s_max = reinterpret_cast<float*>(s_out);  // [2, NW, ER]
        float tg = 0.f, tu = 0.f;
#pragma unroll
        for (int k = 0; k < NI; ++k)
#pragma unroll
          for (int v = 0; v < 8; ++v) {
            const bool real = n0 + 16 * (NI * wn + k) + 8 * (v >> 2) + 4 * e_half + (v & 3) < g.N;
            if (!real) lo[k][v] = hi[k][v] = 0.f;
            tg = fmaxf(tg, finite_abs(lo[k][v]));
            tu = fmaxf(tu, finite_abs(hi[k][v]));
          }
        tg = fmaxf(tg, __shfl_xor(tg, 32, 64));
        tu = fmaxf(tu, __shfl_xor(tu, 32, 64));
        s_max[(e_half * NW + wn) * T::ER + row] = e_half ? tu : tg;
        lds_barrier();
        tg = tu = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          tg = fmaxf(tg, s_max[w * T::ER + row]);
          tu = fmaxf(tu, s_max[(NW + w) * T::ER + row]);
        }
        lds_barrier();  // out goes to the same place
        const int eg = e8m0_of(tg), eu = e8m0_of(tu);
        const float ig = inv_scale(eg), iu = inv_scale(eu);
        if (wn == 0 && 32 * i + e_l32 < mine) {
          const int64_t m = t.m_beg + 32 * (MI * wm + i) + e_l32, nb = g.hs / 128;
          g.kept_s[(2 * m + e_half) * nb + t.nt] = (uint8_t)(e_half ? eu : eg);
        }
#pragma unroll
        for (int k = 0; k < NI; ++k)
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const int c = 16 * (NI * wn + k) + 8 * q + 4 * e_half;  // of the 128 columns
            const float a[4] = {lo[k][4 * q], lo[k][4 * q + 1], lo[k][4 * q + 2], lo[k][4 * q + 3]};
            const float b[4] = {hi[k][4 * q], hi[k][4 * q + 1], hi[k][4 * q + 2], hi[k][4 * q + 3]};
            uint8_t* const to = s_kept + row * T::KEPT_ROW;
            *reinterpret_cast<uint32_t*>(to + 16 * ((c >> 4) ^ (row & 7)) + (c & 15)) = to_codes(a, ig);
            *reinterpret_cast<uint32_t*>(to + 128 + 16 * ((c >> 4) ^ (row & 7)) + (c & 15)) = to_codes(b, iu);
          }
      }
      if (!PARTS || g.parts == 1)
#pragma unroll
      for (int k = 0; k < NI; ++k)
#pragma unroll
        for (int r0 = 0; r0 < VH; r0 += RL) {
          const int v = VH * (KW > 1 ? kw : 0) + r0, c16 = 8 * (v >> 2) + 4 * e_half + (v & 3), b = NI * wn + k;
          if constexpr (!GATED) {
            put(s_out, T::OUT_ROW, row, 32 * b + c16, &lo[k][r0]);
            put(s_out, T::OUT_ROW, row, 32 * b + 16 + c16, &hi[k][r0]);
          } else {
            float a[RL];
#pragma unroll
            for (int x = 0; x < RL; ++x) a[x] = silu_fast(lo[k][r0 + x]) * hi[k][r0 + x];
            put(s_out, T::OUT_ROW, row, 16 * b + c16, a);
            if constexpr (EPI == LIN_GATED) {
              if (g.kept) {
                put(s_kept, T::KEPT_ROW / 2, 2 * row, 16 * b + c16, &lo[k][r0]);
                put(s_kept, T::KEPT_ROW / 2, 2 * row + 1, 16 * b + c16, &hi[k][r0]);
              }
            }
          }
        }
      }
      if (PARTS && g.parts > 1) continue;  // block-uniform
      lds_barrier();
      constexpr int CH = T::OUT_ROW / 16;  // chunks of a row
      const bool vec = g.ldo % 8 == 0 && ((uintptr_t)g.out & 15) == 0;
      for (int at = tid_now; at < T::ER * CH; at += THREADS) {
        const int r = at / CH, c = at % CH, slot = 32 * (MI * (T::EW * h + (r >> 5)) + i) + (r & 31);
        const int64_t n = n0 + 8 * c;
        if (slot < t.valid && n < g.N) {
          const u32x4 v = *reinterpret_cast<const u32x4*>(s_out + r * T::OUT_ROW + 16 * (c ^ (r & (CH - 1))));
          uint16_t* const to = g.out + (t.m_beg + slot) * g.ldo + n;
          if (vec && n + 8 <= g.N) {  // (past the operands in the caches: 8,192 x 14,336 x 4,096 790 -> 768 us)
            __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(to));
          } else {
#pragma unroll
            for (int x = 0; x < 8; ++x)
              if (n + x < g.N) to[x] = (uint16_t)(v[x >> 1] >> (16 * (x & 1)));
          }
        }
      }
      if constexpr (EPI == LIN_GATED) {
        if (g.kept) {
          for (int at = tid_now; at < 2 * T::ER * CH; at += THREADS) {  // rows 2 r (gate) and 2 r + 1 (up)
            const int rr = at / CH, c = at % CH, r = rr >> 1, slot = 32 * (MI * (T::EW * h + (r >> 5)) + i) + (r & 31);
            const int64_t n = n0 + 8 * c;
            if (slot < t.valid && n < g.N)
              __builtin_nontemporal_store(
                  *reinterpret_cast<const u32x4*>(s_kept + rr * (T::KEPT_ROW / 2) + 16 * (c ^ (rr & (CH - 1)))),
                  reinterpret_cast<u32x4*>(reinterpret_cast<uint16_t*>(g.kept) + (2 * (t.m_beg + slot) + (rr & 1)) * g.hs + n));
          }
        }
      } else if constexpr (EPI == LIN_CK8) {
        for (int at = tid_now; at < T::ER * 16; at += THREADS) {
          const int r = at >> 4, c = at & 15, slot = 32 * (MI * (T::EW * h + (r >> 5)) + i) + (r & 31);
          if (slot < t.valid)
            __builtin_nontemporal_store(
                *reinterpret_cast<const u32x4*>(s_kept + r * T::KEPT_ROW + 128 * (c >> 3) + 16 * ((c & 7) ^ (r & 7))),
                reinterpret_cast<u32x4*>(reinterpret_cast<uint8_t*>(g.kept) + (2 * (t.m_beg + slot) + (c >> 3)) * g.hs + n0 +
                                         16 * (c & 7)));
        }
      }
    }
  }
  wait_vmcnt<0>();  // no DMA lands in LDS that is someone else's by then
}

inline bool raise_linear_lds(const void* kernel, size_t bytes) {
  (void)hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  (void)hipGetLastError();
  return true;
}

// One kernel: launch and one-time set-up.
template <int WAVES, int MW, int NW, int MI, int NI, bool Q4, int EPI, int TR = 0>
struct LinLaunch {
  typedef LinTile<WAVES, MW, NW, MI, NI, Q4, EPI> T;
  template <int DT>
  static void prepare_one() {
    static const bool done =
        raise_linear_lds(reinterpret_cast<const void*>(&linear_kernel<WAVES, MW, NW, MI, NI, DT, Q4, EPI, TR>), T::LDS);
    (void)done;
  }
  static void prepare() {
    prepare_one<USAF_BF16>();
    prepare_one<USAF_F16>();
  }
  static int launch(LinArgs g, int dt, hipStream_t st) {
    const int64_t n_nt = (g.N + T::COLS - 1) / T::COLS, units = (g.M + T::M - 1) / T::M * n_nt * g.parts;
    const int64_t cus = device_cu_count();
    if (units >= (int64_t)1 << 30) return set_error(USAF_ERR_UNSUPPORTED, "linear: too many tiles");
    g.n_nt = (int)n_nt;
    const unsigned blocks = (unsigned)(((units < cus ? units : cus) + L_XCDS - 1) / L_XCDS * L_XCDS);
    prepare();
    if (dt == USAF_BF16) linear_kernel<WAVES, MW, NW, MI, NI, USAF_BF16, Q4, EPI, TR><<<blocks, 64 * WAVES, T::LDS, st>>>(g);
    else linear_kernel<WAVES, MW, NW, MI, NI, USAF_F16, Q4, EPI, TR><<<blocks, 64 * WAVES, T::LDS, st>>>(g);
    return check_launch("linear");
  }
};

// Microseconds of a call: rounds of tiles over the CUs, the last one whole, and a launch.  The parts' fp32 sums are
// written and read at about 4 TB/s, in one more launch.  Measured (us, with parts where the rule takes them / without, 4-bit bf16):
// 32 and 100 rows of 14,336 to 4,096 20.8 / 28.0 and 30.3 / 50.1, 32 and 300 of 8,192 to 1,024 11.4 / 16.9 and 22.8 / 29.9,
// 1,000 of 16,384 to 2,048 88.6 / 103.4; 2,048 of them 161.5 / 162.7.
template <class T, int STEP, int END>
double lin_us(const LinArgs& g, bool gated, int parts) {
  const int64_t steps = (g.K / 64 + T::KW - 1) / T::KW, cols = gated ? T::N / 2 : T::N;
  const int64_t tiles = (g.M + T::M - 1) / T::M * ((g.N + cols - 1) / cols) * parts, cus = device_cu_count();
  const double tile = 0.01 * ((double)((steps + parts - 1) / parts) * STEP + END);
  return 3 + tile * (double)((tiles + cus - 1) / cus) + (parts > 1 ? 3 + (double)parts * (double)g.M * (double)g.N * 8 / 4e6 : 0);
}

// One shape of tile for all that leaves it.  FOUR: the plain product of the whole contraction on four waves (2 x 2 of them)
// instead of eight.  STEP: what a step of KW blocks of 64 takes, END: what a tile takes beside its steps, in 10 ns.
template <int MW, int NW, int MI, int NI, bool Q4, int STEP, int END, bool FOUR = false>
struct LinShape {
  typedef LinTile<8, MW, NW, MI, NI, Q4, LIN_STORE> T;
  typedef LinLaunch<8, MW, NW, MI, NI, Q4, LIN_STORE> Store;
  typedef LinLaunch<FOUR ? 4 : 8, FOUR ? 2 : MW, FOUR ? 2 : NW, FOUR ? T::M / 64 : MI, FOUR ? T::N / 64 : NI, Q4, LIN_STORE> Whole;
  typedef LinLaunch<8, MW, NW, MI, NI, Q4, LIN_GATED> Gated;
  static constexpr bool CK8 = T::N == 256 && T::KW == 1;  // may keep 8-bit blocks
  static constexpr int KW = T::KW;

  static void prepare() {
    Store::prepare();
    Whole::prepare();
    Gated::prepare();
    if constexpr (CK8) LinLaunch<8, MW, NW, MI, NI, Q4, LIN_CK8>::prepare();
  }
  static int launch(const LinArgs& g, int dt, bool gated, hipStream_t st) {
    if (!gated) return g.parts > 1 ? Store::launch(g, dt, st) : Whole::launch(g, dt, st);
    if constexpr (CK8) {
      if (g.kept && g.kept_s) return LinLaunch<8, MW, NW, MI, NI, Q4, LIN_CK8>::launch(g, dt, st);
    }
    return Gated::launch(g, dt, st);
  }
  static double us(const LinArgs& g, bool gated, int parts) { return lin_us<T, STEP, END>(g, gated, parts); }
};

// The same for products whose weights (TR = 1) or both operands (2) are stored with the contraction's index first: C = A W,
// C = A^T W.  Their lines of 512 or 256 bytes are a tile's columns of a row; the fragments are read turned out of LDS, at the
// steps' times of the others (2,048 x 2,048 of 16,384 136 to 157 us, 16,384 x 2,048 of 2,048 128 to 140, with the copies' product alike).
template <int MW, int NW, int MI, int NI, int TR, int STEP, int END, bool FOUR = false>
struct LinTurned {
  typedef LinTile<8, MW, NW, MI, NI, false, LIN_STORE> T;
  typedef LinLaunch<8, MW, NW, MI, NI, false, LIN_STORE, TR> Store;
  typedef LinLaunch<FOUR ? 4 : 8, FOUR ? 2 : MW, FOUR ? 2 : NW, FOUR ? T::M / 64 : MI, FOUR ? T::N / 64 : NI, false, LIN_STORE, TR> Whole;
  static constexpr bool CK8 = false;
  static constexpr int KW = T::KW;
  static void prepare() {
    Store::prepare();
    Whole::prepare();
  }
  static int launch(const LinArgs& g, int dt, bool, hipStream_t st) {
    return g.parts > 1 ? Store::launch(g, dt, st) : Whole::launch(g, dt, st);
  }
  static double us(const LinArgs& g, bool, int parts) { return lin_us<T, STEP, END>(g, false, parts); }
};

template <class S>
void consider(LinPlan& best, const LinArgs& g, bool gated) {
  if (gated && g.kept && g.kept_s && !S::CK8) return;
  for (int parts = 1; parts <= (gated ? 1 : 16); parts *= 2) {
    if (parts > 1 && g.K / 64 < 4 * parts * S::KW) break;
    const double us = S::us(g, gated, parts);
    if (best.launch == nullptr || us < best.us) best = {S::launch, parts, us, S::T::M, S::T::N};
  }
}

}  // namespace
}  // namespace usaf

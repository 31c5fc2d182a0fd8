// Matrix products of FP8 codes with a scale for each block of 128 contracted elements:
//
//   y[s][n] = sum over blocks b of  sx[s][b] sw[n / 128][b] * sum_{k in b} x[s][k] w[n][k]
//
// sx is of the row (or of its 128 rows), sw of 128 columns. One matrix instruction of
// depth 128 sums a block, from zero, and a multiplication and addition by the vector units
// puts it to the tile's sums, in float32: four of those for a product of 32 cycles, which
// hide behind it.
//
// The FP8 instructions of gfx950 (of depth 32 as of 128) sum the products of eight
// neighbours with the bits below 2^-13 of the largest one's power of two cut off, and then
// these sums in float32: measured with two products at a time of all distances. Seven of
// eight lose less than 2^-13 of the largest each, 7 2^-13 sum |x w| in all at most; measured
// 1e-5 of that sum for normal values and 7e-5 for ones of widely different sizes. Where
// products do not cancel that is well below the rounding of a 16-bit result, which is what
// it is used for. A float32 result is the sum of exact products instead (EXACT): codes
// become bfloat16, which holds them all, and four instructions of depth 32 sum a block.
//
// Everything else is as in tile_product.hpp: a step is 128 bytes of a row,
// so a block; tiles of LDS filled straight from memory, two steps ahead; Q (the weights) is
// the first operand, so that a lane has one row s, whose scale it multiplies with.
#pragma once

#include "tile_product.hpp"

namespace cck {

// A row of codes; kBytes as RowOperand counts.
struct ElemFP8 {
  static constexpr int kBytes = 1;
  static constexpr bool kScaled = false;
};

constexpr int kBlockStep = 128;

// The operand format of a matrix instruction.
template <int FMT>
constexpr int kOperandFormat = FMT == kF8E4M3 ? 0 : 1;

// A lane's 32 codes of a block, as they are multiplied.
template <int FMT, bool EXACT>
struct BlockFragment {
  u32x4 w[EXACT ? 4 : 2];
  __device__ BlockFragment() = default;
  __device__ BlockFragment(const u32x4& a, const u32x4& b) {
    if constexpr (EXACT) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        w[i / 2][i % 2 * 2] = two(a[i], false);
        w[i / 2][i % 2 * 2 + 1] = two(a[i], true);
        w[2 + i / 2][i % 2 * 2] = two(b[i], false);
        w[2 + i / 2][i % 2 * 2 + 1] = two(b[i], true);
      }
    } else {
      w[0] = a;
      w[1] = b;
    }
  }
  // Two codes as bfloat16.
  __device__ static uint32_t two(uint32_t v, bool high) {
    if constexpr (FMT == kF8E4M3) {
      return __builtin_bit_cast(uint32_t, high ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v, 1.0f, true)
                                               : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v, 1.0f, false));
    } else {
      return __builtin_bit_cast(uint32_t, high ? __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(v, 1.0f, true)
                                               : __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(v, 1.0f, false));
    }
  }
};

template <int FX, int FW, bool EXACT>
__device__ inline f32x4 block_mma(const BlockFragment<FW, EXACT>& w, const BlockFragment<FX, EXACT>& x) {
  const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
  if constexpr (EXACT) {
    f32x4 c = zero;
#pragma unroll
    for (int i = 0; i < 4; ++i) c = ElemBF16::mma(w.w[i], x.w[i], c, 0, 0);
    return c;
  } else {
    i32x8 a, b;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      a[i] = (int)w.w[i / 4][i % 4];
      b[i] = (int)x.w[i / 4][i % 4];
    }
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, zero, kOperandFormat<FW>, kOperandFormat<FX>, 0, 0,
                                                            0, 0);
  }
}
__device__ inline void add_scaled(f32x4& acc, const f32x4& part, float scale) {
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i] = __builtin_fmaf(part[i], scale, acc[i]);
}

struct BlockArgs {
  RowsArgs rows;
  const float *x_scale, *w_scale;
  int blocks, x_shift;  // x_shift: 7 if 128 rows of x share a scale, else 0
  int out_dtype;
};

// fn(codec) of the output: float32 if EXACT, else a 16-bit type.
template <bool EXACT, class Fn>
__device__ inline void with_out(int dtype, Fn&& fn) {
  if constexpr (EXACT) {
    fn(CodecF32{});
  } else if (dtype == kBF16) {
    fn(CodecBF16{});
  } else {
    fn(CodecF16{});
  }
}

// Which rows and columns a workgroup has: as rows_product's.
template <int BP, int BQ, int THREADS>
struct BlockTile {
  RowTileAt at;
  int col, width;
  bool none = false;
  __device__ BlockTile(typename RowTiles<BP, THREADS>::Shared& shared, const RowsArgs& a) {
    int tp, tq;
    const int id = a.first + (int)blockIdx.x;
    if (a.offsets != nullptr) {
      const RowTiles<BP, THREADS> tiles(shared, a.offsets, a.groups, a.rows, a.most);
      const int total = tiles.total * a.tiles_q;
      none = id >= total;
      if (none) return;
      tile_order(xcd_contiguous(id, total), tiles.total, a.tiles_q, &tp, &tq);
      at = tiles.at(tp);
      none = at.count == 0;
    } else {
      tile_order(xcd_contiguous(id, a.most * a.tiles_q), a.most, a.tiles_q, &tp, &tq);
      at.row = (int64_t)tp * BP;
      at.count = a.rows - at.row < BP ? (int)(a.rows - at.row) : BP;
      at.group = 0;
    }
    col = tq * BQ;
    width = a.cols - col < BQ ? a.cols - col : BQ;
  }
};

// Scales of a step in LDS, straight from memory: a word of each row of the tile, then
// one of each 128 columns. A wave asks for 64 words.
template <int BP, int BQ, int NW>
struct BlockScales {
  static constexpr int kRowWaves = BP / 64;
  static_assert(BP % 64 == 0 && kRowWaves < NW);
  static constexpr int kLds = NW * 256;
  const char* base;
  uint32_t off;
  int left;  // blocks

  __device__ BlockScales(const BlockArgs& a, const RowTileAt& at, int col, int width) : left(a.blocks) {
    const int wave = wave_of<NW>(), lane = (int)threadIdx.x & 63;
    const int64_t ld = (int64_t)a.blocks * 4;
    if (wave < kRowWaves) {
      const int64_t first = at.row >> a.x_shift;
      const int row = wave * 64 + lane < at.count ? wave * 64 + lane : at.count - 1;
      base = reinterpret_cast<const char*>(a.x_scale) + first * ld;
      off = (uint32_t)(((at.row + row) >> a.x_shift) - first) * (uint32_t)ld;
    } else {
      const int64_t tall = (a.rows.cols + 127) / 128, first = at.group * tall + col / 128;
      const int most = (width + 127) / 128 - 1, block = (wave - kRowWaves) * 64 + lane;
      base = reinterpret_cast<const char*>(a.w_scale) + first * ld;
      off = (uint32_t)(block < most ? block : most) * (uint32_t)ld;
    }
    base = reinterpret_cast<const char*>(uniform((int64_t)base));
  }
  __device__ void ask(LdsPtr to) {
    lds_place(to + wave_of<NW>() * 256);
    place_ready();
    load_to_place<4, false>(buffer_from(base), left > 0 ? off : kOutOfRange);
    base = in_scalars(base + 4);
    --left;
  }
  __device__ static float row(LdsPtr slot, int r) { return lds_load<float>(slot + r * 4); }
  __device__ static float cols(LdsPtr slot, int c) { return lds_load<float>(slot + kRowWaves * 256 + c / 128 * 4); }
};

template <int FX, int FW, bool EXACT, int WP, int WQ, int FP, int FQ>
__global__ __launch_bounds__(WP* WQ * 64, 2) void block_product(BlockArgs a) {
  constexpr int BP = WP * FP * 16, BQ = WQ * FQ * 16, NW = WP * WQ;
  constexpr bool kPerm = FQ % 4 == 0;
  using P = RowOperand<ElemFP8, BP, NW, false, kBlockStep>;
  using Q = RowOperand<ElemFP8, BQ, NW, kPerm, kBlockStep>;
  using S = BlockScales<BP, BQ, NW>;
  constexpr int kAtQ = P::kLds, kAtS = kAtQ + Q::kLds, kSlot = kAtS + S::kLds, kLds = 2 * kSlot;
  constexpr int kAll = P::kLoads + Q::kLoads + 1;
  static_assert(FQ * 16 <= 128 && 128 % (FQ * 16) == 0);  // a wave's columns share a scale
  // A wave has kAhead columns' codes in registers: behind the products of column j it reads column j + kAhead, of this
  // step or the next one, and behind those of the last one the next step's rows, so that a step begins with what it
  // needs. Behind the products of column kLast the waves meet, once a step: this slot has been read, and the next one
  // has landed. The loads of the step after that go out between the products that are left: at once they would hold
  // each other up, with the matrix cores idle. 8192 rows, 14336 x 4096, us: 419, and with 16384 products a sum 1543; a
  // step's first codes read when it begins 426 and 1600, loads at once 460, a second meeting 445. Two columns ahead in
  // place of four 436 and 1600.
  constexpr int kAhead = FQ == 8 ? 4 : 2, kLast = FQ - kAhead;
  __shared__ __attribute__((aligned(1024))) char lds[kLds];
  __shared__ typename RowTiles<BP, NW * 64>::Shared shared;

  const BlockTile<BP, BQ, NW * 64> tile(shared, a.rows);
  if (tile.none) return;
  const RowTileAt at = tile.at;
  const int wave = wave_of<NW>(), p0 = (wave / WQ) * FP * 16, q0 = (wave % WQ) * FQ * 16;
  const int64_t cols = a.rows.cols;
  const int64_t first_out = at.row * cols + tile.col;
  if (at.group < 0) {
    with_out<EXACT>(a.out_dtype, [&](auto c) {
      using C = decltype(c);
      store_zeros<C, NW>(a.rows.out + first_out * C::kBytes, cols, at.count, tile.width);
    });
    return;
  }
  const int64_t ld = a.rows.length;
  P p(a.rows.x + at.row * ld, ld, at.count, ld);
  Q q(a.rows.w + ((int64_t)at.group * cols + tile.col) * ld, ld, tile.width, ld);
  S s(a, at, tile.col, tile.width);
  const LdsPtr slots = (LdsPtr)lds;
  // Load i of a step.
  auto ask_one = [&](LdsPtr to, int i) __attribute__((always_inline)) {
    if (i < P::kLoads) {
      P::place(to, i);
      place_ready();
      p.fetch(i);
    } else if (i < P::kLoads + Q::kLoads) {
      Q::place(to + kAtQ, i - P::kLoads);
      place_ready();
      q.fetch(i - P::kLoads);
    } else {
      s.ask(to + kAtS);
    }
  };
  auto ask = [&](LdsPtr to, int begin, int end) __attribute__((always_inline)) {
#pragma unroll
    for (int i = begin; i < end; ++i) ask_one(to, i);
  };
  auto advance = [&] {
    p.advance();
    q.advance();
  };
  const bool live = p0 < at.count && q0 < tile.width;
  const typename P::template Lane<FP> p_lane(slots, p0);
  const typename Q::template Lane<FQ> q_lane(slots + kAtQ, q0);
  const int lane = (int)threadIdx.x & 63;
  f32x4 acc[FP][FQ] = {};
  ask(slots, 0, kAll);
  advance();
  ask(slots + kSlot, 0, kAll);
  advance();
  loads_landed<kAll>();
  meet();
  u32x4 x[FP][2], w[kAhead][2];
  BlockFragment<FX, EXACT> wide[FP];  // EXACT: x, once a step
  float scale[FP], next[FP], of_cols = 0.0f;
  f32x4 part[FP];
  auto read_x = [&](int i, int slot) __attribute__((always_inline)) {
    x[i][0] = p_lane.fragment(i, 0, slot);
    x[i][1] = p_lane.fragment(i, 1, slot);
    next[i] = S::row(slots + slot + kAtS, p0 + 16 * i + (lane & 15));
  };
  auto read_w = [&](int j, int slot) __attribute__((always_inline)) {
    w[j % kAhead][0] = q_lane.fragment(j, 0, slot);
    w[j % kAhead][1] = q_lane.fragment(j, 1, slot);
  };
  if (live) {
#pragma unroll
    for (int j = 0; j < kAhead; ++j) read_w(j, 0);
#pragma unroll
    for (int i = 0; i < FP; ++i) {
      read_x(i, 0);
      scale[i] = 0.0f;
      part[i] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    }
    of_cols = S::cols(slots + kAtS, q0);
  }
  for (int t = 0; t < a.blocks; ++t) {
    const int slot = (t & 1) * kSlot, other = kSlot - slot;
    const LdsPtr now = slots + slot;
    if (live) {
#pragma unroll
      for (int j = 0; j < FQ; ++j) {
        const BlockFragment<FW, EXACT> column(w[j % kAhead][0], w[j % kAhead][1]);
#pragma unroll
        for (int i = 0; i < FP; ++i) {
          // Each product is added FP products later, when the matrix cores are done with it.
          add_scaled(acc[i][j == 0 ? FQ - 1 : j - 1], part[i], scale[i]);
          if (j == 0) {
            scale[i] = next[i] * of_cols;
            if (EXACT) wide[i] = BlockFragment<FX, EXACT>(x[i][0], x[i][1]);
          }
          part[i] = block_mma<FX, FW, EXACT>(column, EXACT ? wide[i] : BlockFragment<FX, EXACT>(x[i][0], x[i][1]));
          if (j == FQ - 1) read_x(i, other);
          if (j > kLast) {
            constexpr int kSpread = (FQ - 1 - kLast) * FP;
            const int n = (j - kLast - 1) * FP + i;
            ask(now, n * kAll / kSpread, (n + 1) * kAll / kSpread);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        if (j == kLast) {
          lds_read();
          loads_landed();
          meet();
        }
        read_w((j + kAhead) % FQ, j < kLast ? slot : other);
        if (j == FQ - 1) of_cols = S::cols(slots + other + kAtS, q0);
      }
    } else {
      loads_landed();
      meet();
      ask(now, 0, kAll);
    }
    advance();
  }
  if (live) {
#pragma unroll
    for (int i = 0; i < FP; ++i) add_scaled(acc[i][FQ - 1], part[i], scale[i]);
  }
  loads_landed();
  meet();  // nobody reads the slots any more, and nothing is on its way to them
  if (!live) return;
  with_out<EXACT>(a.out_dtype, [&](auto c) {
    using C = decltype(c);
    store_tile<C, kPerm, FP, FQ, kLds / NW / 1024 * 1024>(acc, slots + wave * (kLds / NW / 1024 * 1024),
                                                          a.rows.out + first_out * C::kBytes, cols, p0, q0, at.count,
                                                          tile.width);
  });
}

// Rows of any length and alignment (16 bytes or more): loads wait in registers for a step,
// and scales come straight to them. 1554 rows on 8 experts of 1412 x 1030, float32 results, 18 us:
// nine steps of 1.4 us, by the reads of 64 x 64 tiles from L2, off their lines (3 us less for
// 1024), and 5 us beside them. Loads two steps ahead took as long. It is the one kernel for
// such rows, few or many: dense bf16 results, us, and of whole vectors 4096 long: 8 rows,
// 14336 x 4095 43 and 13; 8192 rows 2086 and 456; 8192 rows, 4096 x 4095 605 and 135.
template <int FX, int FW, bool EXACT, int WP, int WQ, int FP, int FQ>
__global__ __launch_bounds__(WP* WQ * 64, 2) void block_product_ragged(BlockArgs a) {
  constexpr int BP = WP * FP * 16, BQ = WQ * FQ * 16, NW = WP * WQ;
  constexpr bool kPerm = FQ % 4 == 0;
  using P = RowOperand<ElemFP8, BP, NW, false, kBlockStep>;
  using Q = RowOperand<ElemFP8, BQ, NW, kPerm, kBlockStep>;
  constexpr int kAtQ = P::kLds, kSlot = kAtQ + Q::kLds, kLds = 2 * kSlot;
  __shared__ __attribute__((aligned(1024))) char lds[kLds];
  __shared__ typename RowTiles<BP, NW * 64>::Shared shared;

  const BlockTile<BP, BQ, NW * 64> tile(shared, a.rows);
  if (tile.none) return;
  const RowTileAt at = tile.at;
  const int wave = wave_of<NW>(), p0 = (wave / WQ) * FP * 16, q0 = (wave % WQ) * FQ * 16;
  const int64_t cols = a.rows.cols;
  const int64_t first_out = at.row * cols + tile.col;
  if (at.group < 0) {
    with_out<EXACT>(a.out_dtype, [&](auto c) {
      using C = decltype(c);
      store_zeros<C, NW>(a.rows.out + first_out * C::kBytes, cols, at.count, tile.width);
    });
    return;
  }
  const int64_t ld = a.rows.length;
  P p(a.rows.x + at.row * ld, ld, at.count, ld);
  Q q(a.rows.w + ((int64_t)at.group * cols + tile.col) * ld, ld, tile.width, ld);
  const LdsPtr slots = (LdsPtr)lds;
  const bool live = p0 < at.count && q0 < tile.width;
  const typename P::template Lane<FP> p_lane(slots, p0);
  const typename Q::template Lane<FQ> q_lane(slots + kAtQ, q0);
  const float* x_scale[FP];
#pragma unroll
  for (int i = 0; i < FP; ++i) {
    const int row = p0 + 16 * i + ((int)threadIdx.x & 15);
    x_scale[i] = a.x_scale + ((at.row + (row < at.count ? row : at.count - 1)) >> a.x_shift) * a.blocks;
  }
  const int col = live ? tile.col + q0 : tile.col;
  const float* w_scale = a.w_scale + ((int64_t)at.group * ((cols + 127) / 128) + col / 128) * a.blocks;
  u32x4 held_p[P::kLoads], held_q[Q::kLoads];
  f32x4 acc[FP][FQ] = {};
  p.load(held_p);
  q.load(held_q);
  for (int t = 0; t < a.blocks; ++t) {
    const int slot = (t & 1) * kSlot;
    p.store(held_p, slots + slot, 0);
    q.store(held_q, slots + slot + kAtQ, 0);
    __syncthreads();
    if (t + 1 < a.blocks) {
      p.advance();
      q.advance();
      p.load(held_p);
      q.load(held_q);
    }
    if (live) {
      BlockFragment<FX, EXACT> x[FP];
      float scale[FP];
      const float of_cols = w_scale[t];
#pragma unroll
      for (int i = 0; i < FP; ++i) {
        x[i] = BlockFragment<FX, EXACT>(p_lane.fragment(i, 0, slot), p_lane.fragment(i, 1, slot));
        scale[i] = x_scale[i][t] * of_cols;
      }
#pragma unroll
      for (int j = 0; j < FQ; ++j) {
        const BlockFragment<FW, EXACT> w(q_lane.fragment(j, 0, slot), q_lane.fragment(j, 1, slot));
#pragma unroll
        for (int i = 0; i < FP; ++i) add_scaled(acc[i][j], block_mma<FX, FW, EXACT>(w, x[i]), scale[i]);
      }
    }
  }
  __syncthreads();  // nobody reads the slots any more
  if (!live) return;
  with_out<EXACT>(a.out_dtype, [&](auto c) {
    using C = decltype(c);
    store_tile<C, kPerm, FP, FQ, kLds / NW>(acc, slots + wave * (kLds / NW), a.rows.out + first_out * C::kBytes, cols,
                                            p0, q0, at.count, tile.width);
  });
}

// Few rows a group: a workgroup owns FP x 16 rows and FQ x 16 columns, and its waves take
// the blocks in turn, each through a ring of DEPTH steps in LDS that it keeps to itself.
// The sums of the waves meet in LDS at the end, in the order of the waves. Bound by HBM, the
// weights: 8 rows, 14336 x 4096, 59 MB, 10.9 us, 5.4 TB/s, of which the ramp is a part.
template <int FX, int FW, bool EXACT, int FP, int FQ, int NW, int DEPTH>
__global__ __launch_bounds__(NW * 64, 2) void block_stream(BlockArgs a) {
  constexpr int BP = FP * 16, BQ = FQ * 16;
  using P = RowOperand<ElemFP8, BP, 1, false, kBlockStep>;
  using Q = RowOperand<ElemFP8, BQ, 1, false, kBlockStep>;
  constexpr int kAtQ = P::kLds, kAtS = kAtQ + Q::kLds, kSlot = kAtS + 512, kRing = DEPTH * kSlot;
  constexpr int kSums = NW * FP * FQ * 1024, kAll = P::kLoads + Q::kLoads + 2;
  static_assert(BP <= 64 && 128 % BQ == 0 && (DEPTH - 1) * kAll < 64);
  __shared__ __attribute__((aligned(1024))) char lds[NW * kRing > kSums ? NW * kRing : kSums];
  __shared__ typename RowTiles<BP, NW * 64>::Shared shared;

  const BlockTile<BP, BQ, NW * 64> tile(shared, a.rows);
  if (tile.none) return;
  const RowTileAt at = tile.at;
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int64_t cols = a.rows.cols, ld = a.rows.length;
  f32x4 acc[FP][FQ] = {};
  if (at.group >= 0) {
    const LdsPtr ring = (LdsPtr)lds + wave * kRing;
    P p(a.rows.x + at.row * ld, ld, at.count, ld);
    Q q(a.rows.w + ((int64_t)at.group * cols + tile.col) * ld, ld, tile.width, ld);
    const int64_t first = at.row >> a.x_shift;
    const int row = lane < at.count ? lane : at.count - 1;
    const uint32_t scale_off = (uint32_t)(((at.row + row) >> a.x_shift) - first) * (uint32_t)(a.blocks * 4);
    const char* xs = reinterpret_cast<const char*>(a.x_scale + first * a.blocks + wave);
    const char* ws = reinterpret_cast<const char*>(
        a.w_scale + ((int64_t)at.group * ((cols + 127) / 128) + tile.col / 128) * a.blocks + wave);
    int left = a.blocks - wave;
    p.advance(wave);
    q.advance(wave);
    auto ask = [&](LdsPtr to) __attribute__((always_inline)) {  // a step past the end is zeros
#pragma unroll
      for (int i = 0; i < P::kLoads; ++i) {
        P::place(to, i);
        place_ready();
        p.fetch(i);
      }
#pragma unroll
      for (int i = 0; i < Q::kLoads; ++i) {
        Q::place(to + kAtQ, i);
        place_ready();
        q.template fetch<true>(i);
      }
      lds_place(to + kAtS);
      place_ready();
      load_to_place<4, false>(buffer_from(xs), left > 0 ? scale_off : kOutOfRange);
      lds_place(to + kAtS + 256);
      place_ready();
      load_to_place<4, false>(buffer_from(ws), left > 0 ? 0u : kOutOfRange);
      xs = in_scalars(xs + NW * 4);
      ws = in_scalars(ws + NW * 4);
      left -= NW;
      p.advance(NW);
      q.advance(NW);
    };
    const typename P::template Lane<FP> p_lane(ring, 0);
    const typename Q::template Lane<FQ> q_lane(ring + kAtQ, 0);
    const int steps = (a.blocks - wave + NW - 1) / NW;
    for (int d = 0; d < DEPTH; ++d) ask(ring + d * kSlot);
    int slot = 0;
    for (int t = 0; t < steps; ++t) {
      loads_landed<(DEPTH - 1) * kAll>();
      u32x4 x[FP][2], w[FQ][2];
      float scale[FP];
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
        for (int f = 0; f < FQ; ++f) w[f][ks] = q_lane.fragment(f, ks, slot * kSlot);
#pragma unroll
        for (int f = 0; f < FP; ++f) x[f][ks] = p_lane.fragment(f, ks, slot * kSlot);
      }
      const LdsPtr from = ring + slot * kSlot + kAtS;
#pragma unroll
      for (int f = 0; f < FP; ++f) scale[f] = lds_load<float>(from + (16 * f + (lane & 15)) * 4);
      const float of_cols = lds_load<float>(from + 256);
      lds_read();
      ask(ring + slot * kSlot);
#pragma unroll
      for (int i = 0; i < FP; ++i) {
        const float s = scale[i] * of_cols;
        const BlockFragment<FX, EXACT> row(x[i][0], x[i][1]);
#pragma unroll
        for (int j = 0; j < FQ; ++j) {
          add_scaled(acc[i][j], block_mma<FX, FW, EXACT>(BlockFragment<FW, EXACT>(w[j][0], w[j][1]), row), s);
        }
      }
      slot = slot + 1 < DEPTH ? slot + 1 : 0;
    }
    loads_landed();
  }
  f32x4* const part = reinterpret_cast<f32x4*>(lds) + lane;  // [NW][FP * FQ][64]
  __syncthreads();  // the rings are read
#pragma unroll
  for (int i = 0; i < FP; ++i) {
#pragma unroll
    for (int j = 0; j < FQ; ++j) part[(wave * FP * FQ + i * FQ + j) * 64] = acc[i][j];
  }
  __syncthreads();
  for (int f = wave; f < FP * FQ; f += NW) {
    f32x4 sum = part[f * 64];
#pragma unroll
    for (int w = 1; w < NW; ++w) sum += part[(w * FP * FQ + f) * 64];
    with_out<EXACT>(a.out_dtype, [&](auto c) {
      using C = decltype(c);
      store_fragment<C>(sum, a.rows.out + (at.row * cols + tile.col) * C::kBytes, cols, 16 * (f / FQ), 16 * (f % FQ),
                        at.count, tile.width);
    });
  }
}

// Rows of fewer than 16 codes: an element of the output a thread.
template <int FX, int FW, bool EXACT>
__global__ __launch_bounds__(256) void block_narrow(BlockArgs a) {
  const RowsArgs& r = a.rows;
  const int64_t total = r.rows * r.cols;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / r.cols, col = i - row * r.cols;
    int64_t group = 0;
    if (r.offsets != nullptr) {
      int lo = 0, hi = r.groups + 1;  // offsets[lo - 1] <= row < offsets[hi], of those that are in order
      while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (r.offsets[mid] <= row) {
          lo = mid + 1;
        } else {
          hi = mid;
        }
      }
      group = lo >= 1 && lo <= r.groups ? lo - 1 : -1;
    }
    float sum = 0.0f;
    if (group >= 0) {
      const uint8_t* x = reinterpret_cast<const uint8_t*>(r.x) + row * r.length;
      const uint8_t* w = reinterpret_cast<const uint8_t*>(r.w) + (group * r.cols + col) * r.length;
      for (int k = 0; k < (int)r.length; ++k) {
        const float u = FX == kF8E4M3 ? __builtin_amdgcn_cvt_f32_fp8((int)x[k], 0) : __builtin_amdgcn_cvt_f32_bf8((int)x[k], 0);
        const float v = FW == kF8E4M3 ? __builtin_amdgcn_cvt_f32_fp8((int)w[k], 0) : __builtin_amdgcn_cvt_f32_bf8((int)w[k], 0);
        sum = __builtin_fmaf(u, v, sum);
      }
      sum *= a.x_scale[row >> a.x_shift] * a.w_scale[group * ((r.cols + 127) / 128) + col / 128];
    }
    with_out<EXACT>(a.out_dtype, [&](auto c) { decltype(c)::store1(r.out, i, sum); });
  }
}

// The grid of `kernel`, whose workgroups of `threads` own BP rows and BQ columns.
template <int BP, int BQ>
int32_t launch_block_grid(void (*kernel)(BlockArgs), int threads, BlockArgs a, hipStream_t st) {
  RowsArgs& r = a.rows;
  const int64_t edges = r.offsets == nullptr ? 1 : r.groups + 2;  // each group ends inside one tile at most
  int64_t most = (r.rows + edges * (BP - 1)) / BP;
  most = most < r.rows ? most : r.rows;
  r.most = (int)most;
  r.tiles_q = (int)(((int64_t)r.cols + BQ - 1) / BQ);
  return launch_tiles(most * r.tiles_q, threads, [&](int first, unsigned count) {
    a.rows.first = first;
    kernel<<<count, threads, 0, st>>>(a);
  });
}

template <int FX, int FW, bool EXACT, int WP, int WQ, int FP, int FQ, bool DIRECT>
int32_t launch_block_tiles(const BlockArgs& a, hipStream_t st) {
  constexpr int kThreads = WP * WQ * 64, BP = WP * FP * 16, BQ = WQ * FQ * 16;
  if constexpr (DIRECT) {
    return launch_block_grid<BP, BQ>(block_product<FX, FW, EXACT, WP, WQ, FP, FQ>, kThreads, a, st);
  } else {
    return launch_block_grid<BP, BQ>(block_product_ragged<FX, FW, EXACT, WP, WQ, FP, FQ>, kThreads, a, st);
  }
}

template <int FX, int FW, bool EXACT, int FP, int FQ, int DEPTH>
int32_t launch_block_stream(const BlockArgs& a, hipStream_t st) {
  return launch_block_grid<FP * 16, FQ * 16>(block_stream<FX, FW, EXACT, FP, FQ, 4, DEPTH>, 256, a, st);
}

// Which kernel. bf16 results, us, weights from HBM; float32 ones go the same ways.
// Streams read the weights once for each 16 or 32 rows, and are for few rows:
//   where they make no more than two workgroups a CU. Streams of 32 rows against 64 x 64 tiles: 4096 x 4096, 128
//   rows (512 workgroups) 12.8 and 14.2, 192 rows 17.4 and 14.5; 1408 x 2048, 256 rows (352) 7.8 and 8.7, 384 rows
//   11.3 and 8.7; 14336 x 4096, 32 rows (448) 16.3 and 17.2, 48 rows 26.0 and 18.1;
//   and for groups of 16 rows or less on average, whose rows are long enough for four waves: 8 of 14336 x 4096, of
//   16 rows 90.8 and 93.1, of 24 rows 98.5 and 95.7; but 64 of 1408 x 2048, of 8 rows 40.5 and 29.2.
// Of 16 rows and two fragments of columns, or one where that leaves CUs without (4096 x 4096, 16 rows 7.4 and 6.9).
// Tiles of 256 x 256 where they are filled and enough for the CUs (against 128 x 128: 14336 x 4096, 1024 rows, 224
// tiles 65.8 and 80.0, 512 rows, 112 tiles 63.3 and 45.8; 8 groups of 512 rows, 2048 x 2048, 160 by this count 31.5
// and 22.5; 8 of 1024 rows, 288 37.4 and 42.4; 64 groups of 128 rows, 1408 x 2048 47.1 and 39.5, which are half empty;
// 8 of 128 rows, 14336 x 4096 116 and 124; of 192 rows 133 and 151); not for float32 results, whose fragments are
// twice as large.
// Tiles of 64 x 64 where there would be fewer than 220 of 128 x 128 (against those: 8 groups of 128 rows, 2048 x 2048,
// 208 by this count 12.2 and 15.4, of 192 rows, 272 16.1 and 15.6; 14336 x 4096, 192 rows, 224 35.3 and 24.2; 1408 x
// 2048, 2048 rows, 187 14.8 and 14.5, 4096 rows, 363 25.2 and 19.7), and for groups that those leave three quarters empty (8 of 32 rows, 14336 x 4096 98.6
// and 102; of 64 rows 116 and 108).
template <int FX, int FW, bool EXACT>
int32_t launch_block_linear(const BlockArgs& a, hipStream_t st) {
  const RowsArgs& r = a.rows;
  if (r.length < 16) {
    const int64_t blocks = (r.rows * r.cols + 255) / 256;
    block_narrow<FX, FW, EXACT><<<(unsigned)(blocks < 65536 ? blocks : 65536), 256, 0, st>>>(a);
    return launch_status();
  }
  const bool whole = r.length % 16 == 0 && host_aligned(r.x, 16) && host_aligned(r.w, 16) && host_aligned(a.x_scale, 4) &&
                     host_aligned(a.w_scale, 4);
  if (!whole) return launch_block_tiles<FX, FW, EXACT, 2, 2, 2, 2, false>(a, st);
  const int64_t groups = r.groups, cols = r.cols;
  // Of all groups, if they are equal.
  const auto row_tiles = [&](int64_t height) {
    const int64_t tiles = groups * ((r.rows + groups * height - 1) / (groups * height));
    return tiles < r.rows ? tiles : r.rows;
  };
  if (r.rows <= 16 * groups) {
    if (row_tiles(16) * ((cols + 31) / 32) <= 512 || a.blocks >= 32) {
      if (row_tiles(16) * cols >= 256 * 32) return launch_block_stream<FX, FW, EXACT, 1, 2, 2>(a, st);
      return launch_block_stream<FX, FW, EXACT, 1, 1, 2>(a, st);
    }
  } else if (row_tiles(32) * ((cols + 31) / 32) <= 512) {
    return launch_block_stream<FX, FW, EXACT, 2, 2, 2>(a, st);
  }
  if constexpr (!EXACT) {
    if (r.rows >= 160 * groups && (r.rows / 256 + groups / 2) * ((cols + 255) / 256) >= 200) {
      return launch_block_tiles<FX, FW, EXACT, 4, 2, 4, 8, true>(a, st);
    }
  }
  if (r.rows > 32 * groups && (r.rows / 128 + groups / 2 + 1) * ((cols + 127) / 128) >= 220) {
    return launch_block_tiles<FX, FW, EXACT, 2, 2, 4, 4, true>(a, st);
  }
  return launch_block_tiles<FX, FW, EXACT, 2, 2, 2, 2, true>(a, st);
}

}  // namespace cck

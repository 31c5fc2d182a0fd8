// Matrix products grouped by expert, with groups of any size: the linear layers
// of a mixture-of-experts FFN on rows in expert order, and their gradients.
//
//   y[s][n]         = sum_k x[s][k] * w[e][n][k]          launch_grouped_linear_fwd
//   grad_x[s][k]    = sum_n grad_y[s][n] * w[e][n][k]     launch_grouped_linear_grad_input
//   grad_w[e][n][k] = sum_s grad_y[s][n] * x[s][k]        launch_grouped_linear_grad_weight
//
// with e the expert whose rows offsets[e] .. offsets[e + 1] hold s. Products are
// exact in fp32 (fp32 inputs: rounded by the MFMA), sums fp32, and the result is
// rounded once to the storage type. Rows of no expert are zero in y and grad_x,
// and an expert without rows has a zero gradient. The group sizes stay on the
// GPU: the grid has room for the most tiles that `rows` rows can make.
//
// 8192 unevenly routed rows on 8 experts of 14336 x 4096, bf16: 790, 871 and 861 us (1.22,
// 1.10 and 1.12 PFLOP/s), with the matrix cores busy 72, 58 and 60 % of the cycles, at the
// clock that the power limit leaves (1.7 GHz). The loop itself keeps them busy 92, 90 and
// 87 % (see Product). What else there is: a tile's ends, as long as 7 to 9 of its steps (64
// steps in y, 16 on average in grad_w); cut tiles; and in grad_x 2.25 rounds of tiles that
// take three. 16 rows: 113 us, bound by reading the weights.
#include "tile_product.hpp"

namespace cck {
namespace {

// An expert's tiles take as long as it has rows, so every XCD gets a share of each
// expert's where there are enough of them to share (room: up to a multiple of 8, at which
// the next expert begins); else each takes a run of experts. With a run of all tiles each,
// one expert an XCD, eight experts of 8192 unevenly routed rows took 1255 us in place of 864.
constexpr int kTilesApart = 64;
__host__ __device__ constexpr int weights_room(int each) { return each < kTilesApart ? each : (each + 7) / 8 * 8; }

template <class T, class C, int WP, int WQ, int FP, int FQ, bool DIRECT>
__global__ __launch_bounds__(WP* WQ * 64, tile_waves(FP* FQ, DIRECT)) void grouped_weights(
    const char* __restrict__ grad, const char* __restrict__ x, const int64_t* __restrict__ offsets,
    char* __restrict__ out, int64_t rows, int n, int k, int tiles_p, int tiles_q, int first, int total) {
  constexpr int BP = WP * FP * 16, BQ = WQ * FQ * 16, NW = WP * WQ, kStep = DIRECT ? 128 : 64;
  using P = ColOperand<T, BP, NW, kStep>;
  using Q = ColOperand<T, BQ, NW, kStep>;
  using Prod = Product<T, P, Q, NoScales, NoScales, WP, WQ, FP, FQ, kStep>;
  __shared__ __attribute__((aligned(1024))) char lds[Prod::kLds];

  const int each = tiles_p * tiles_q, room = weights_room(each);
  const int id = first + (int)blockIdx.x;
  int e, t;
  if (room >= kTilesApart) {
    e = id / room;
    t = xcd_contiguous(id - e * room, room);
    if (t >= each) return;
  } else {
    t = xcd_contiguous(id, total);
    e = t / each;
    t -= e * each;
  }
  int tp, tq;
  tile_order(t, tiles_p, tiles_q, &tp, &tq);
  const int64_t lo = uniform(clamp_row(offsets[e], rows)), hi = uniform(clamp_row(offsets[e + 1], rows));
  const int64_t length = hi > lo ? hi - lo : 0;
  const int p0 = tp * BP, q0 = tq * BQ;
  const int height = n - p0 < BP ? n - p0 : BP, width = k - q0 < BQ ? k - q0 : BQ;
  P p(grad + (lo * n + p0) * T::kBytes, (int64_t)n * T::kBytes, height, length);
  Q q(x + (lo * k + q0) * T::kBytes, (int64_t)k * T::kBytes, width, length);
  const int steps = (int)((length + P::kDepth - 1) / P::kDepth), wave = wave_of<NW>();
  const int wp0 = (wave / WQ) * FP * 16, wq0 = (wave % WQ) * FQ * 16;
  char* const to = out + (((int64_t)e * n + p0) * k + q0) * C::kBytes;
  if (steps == 0) {
    store_zeros<C, NW>(to, k, height, width);
    return;
  }
  if (wp0 >= height || wq0 >= width) {
    Prod::idle(p, q, NoScales(), NoScales(), steps, (LdsPtr)lds);
    return;
  }
  f32x4 acc[FP][FQ] = {};
  Prod::run(p, q, NoScales(), NoScales(), steps, (LdsPtr)lds, wp0, wq0, acc);
  store_tile<C, false, FP, FQ, Prod::kLds / NW>(acc, (LdsPtr)lds + wave * (Prod::kLds / NW), to, k, wp0, wq0, height,
                                                width);
}

// fn(element type, its storage codec) for a dtype tag.
template <class Fn>
inline int32_t with_elem(int32_t dtype, Fn&& fn) {
  switch (dtype) {
    case kF32: return fn(ElemF32{}, CodecF32{});
    case kF16: return fn(ElemF16{}, CodecF16{});
    case kBF16: return fn(ElemBF16{}, CodecBF16{});
    default: return (int32_t)hipErrorInvalidValue;
  }
}

inline bool whole_vectors(const void* a, const void* b, int64_t n, int64_t k, int64_t bytes) {
  return n * bytes % 16 == 0 && k * bytes % 16 == 0 && host_aligned(a, 16) && host_aligned(b, 16);
}

// y or grad_x: rows of `length` elements against w, rows of `cols` out.
template <bool QROWS>
int32_t grouped_rows(const void* x, const void* w, const int64_t* offsets, void* out, int64_t rows, int64_t groups,
                     int64_t length, int64_t cols, int32_t dtype, void* stream) {
  return with_elem(dtype, [&](auto elem, auto codec) {
    using T = decltype(elem);
    using C = decltype(codec);
    if (rows <= 0 || length < 0 || cols <= 0) return (int32_t)hipSuccess;
    if (!sizes_ok(rows, groups, cols * T::kBytes, length * T::kBytes)) return (int32_t)hipErrorInvalidValue;
    if (length == 0) return launch_zero_rows<C>(out, rows * cols, static_cast<hipStream_t>(stream));
    const RowsArgs a = {static_cast<const char*>(x), static_cast<const char*>(w), nullptr, nullptr, offsets,
                        static_cast<char*>(out), rows, length, (int)groups, (int)cols, 0, 0, 0};
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (length * T::kBytes < 16 || (!QROWS && cols * T::kBytes < 16)) {
      const NarrowArgs n = {a.x, a.w, offsets, a.out, rows, length, 1, QROWS ? length : 1, QROWS ? 1 : cols,
                            length * cols, 0, cols, length, (int)groups};
      narrow_rows<C><<<narrow_grid(rows * cols), 256, 0, st>>>(n);
      return launch_status();
    }
    const bool whole = whole_vectors(x, w, cols, length, T::kBytes);
    if constexpr (QROWS) {
      return whole ? launch_rows_by_size<T, C, true>(a, st) : launch_rows_by_size<T, C, false>(a, st);
    } else {
      if constexpr (T::kAccumulates) {
        if (whole && wide_tiles<T>(a)) return launch_rows<T, C, false, 2, 2, 8, 8, true>(a, st);
      }
      return whole ? launch_rows_small<T, C, false, true>(a, st) : launch_rows_small<T, C, false, false>(a, st);
    }
  });
}

template <class T, class C, int WP, int WQ, int FP, int FQ, bool DIRECT>
int32_t run_weights(const void* grad, const void* x, const int64_t* offsets, void* out, int64_t rows, int64_t groups,
                    int64_t n, int64_t k, hipStream_t st) {
  constexpr int BP = WP * FP * 16, BQ = WQ * FQ * 16, NW = WP * WQ;
  const int64_t tiles_p = (n + BP - 1) / BP, tiles_q = (k + BQ - 1) / BQ;
  if (tiles_p * tiles_q > INT32_MAX - 7) return (int32_t)hipErrorInvalidValue;
  const int64_t total = groups * weights_room((int)(tiles_p * tiles_q));
  return launch_tiles(total, NW * 64, [&](int first, unsigned count) {
    grouped_weights<T, C, WP, WQ, FP, FQ, DIRECT><<<count, NW * 64, 0, st>>>(
        static_cast<const char*>(grad), static_cast<const char*>(x), offsets, static_cast<char*>(out), rows, (int)n,
        (int)k, (int)tiles_p, (int)tiles_q, first, (int)total);
  });
}

// Tiles of 256 x 256 where experts have 768 rows or more on average and each CU gets a tile
// (bf16, us, against 128 x 128: 8 experts of 1024 rows, 2048 x 1408 65.7 and 67.8, of 512 rows,
// 2048 x 2048 49.3 and 46.5; one of 4096 rows, 4096 x 4096 98.9 and 131); of 64 x 64 where
// fewer than 96 of 128 x 128 would share the 256 CUs. bf16, us, 64 x 64 and 128 x 128: 64 tiles
// of 128 x 128, 8192 rows 54.5 and 67.6, of 500 rows 4.9 and 7.4; 96 tiles, one expert of 8192
// rows 55.7 and 67.5, 6 of 1365 rows 15.2 and 14.0, of 500 rows 5.8 and 7.5; 128 tiles, one of
// 8192 rows 57.1 and 69.1, 8 of 1024 rows 14.4 and 11.2, of 500 rows 8.3 and 7.6; 160 tiles,
// one of 8192 rows 93.4 and 68.7, 10 of 819 rows 16.2 and 9.6, of 500 rows 11.5 and 7.6. So
// from 96 to 128 tiles it is the number of experts that decides, which the rule leaves out.
// Always 64 x 64 for fp32 (us, against 128 x 128: 8192 rows, 1024 x 1024 170 and 514; 8 experts
// of 512 rows, 2048 x 1408 186 and 197; one of 4096 rows, 4096 x 4096 989 and 960).
template <class T, class C, bool WHOLE>
int32_t run_weights_by_size(const void* grad, const void* x, const int64_t* offsets, void* out, int64_t rows,
                            int64_t groups, int64_t n, int64_t k, hipStream_t st) {
  if constexpr (T::kBytes != 4) {
    if constexpr (WHOLE) {
      if (rows >= 768 * groups && groups * ((n + 255) / 256) * ((k + 255) / 256) >= 256) {
        return run_weights<T, C, 2, 2, 8, 8, true>(grad, x, offsets, out, rows, groups, n, k, st);
      }
    }
    if (groups * ((n + 127) / 128) * ((k + 127) / 128) >= 96) {
      return run_weights<T, C, 2, 2, 4, 4, WHOLE>(grad, x, offsets, out, rows, groups, n, k, st);
    }
  }
  return run_weights<T, C, 2, 2, 2, 2, WHOLE>(grad, x, offsets, out, rows, groups, n, k, st);
}

}  // namespace
}  // namespace cck

using namespace cck;

extern "C" int32_t launch_grouped_linear_fwd(const void* x, const void* weight, const int64_t* offsets, void* y,
                                             int64_t rows, int64_t num_experts, int64_t n, int64_t k, int32_t dtype,
                                             void* stream) {
  return grouped_rows<true>(x, weight, offsets, y, rows, num_experts, k, n, dtype, stream);
}

extern "C" int32_t launch_grouped_linear_grad_input(const void* grad_y, const void* weight, const int64_t* offsets,
                                                    void* grad_x, int64_t rows, int64_t num_experts, int64_t n,
                                                    int64_t k, int32_t dtype, void* stream) {
  return grouped_rows<false>(grad_y, weight, offsets, grad_x, rows, num_experts, n, k, dtype, stream);
}

extern "C" int32_t launch_grouped_linear_grad_weight(const void* grad_y, const void* x, const int64_t* offsets,
                                                     void* grad_weight, int64_t rows, int64_t num_experts, int64_t n,
                                                     int64_t k, int32_t dtype, void* stream) {
  const hipStream_t st = static_cast<hipStream_t>(stream);
  return with_elem(dtype, [&](auto elem, auto codec) {
    using T = decltype(elem);
    using C = decltype(codec);
    if (num_experts <= 0 || n <= 0 || k <= 0) return (int32_t)hipSuccess;
    if (!sizes_ok(rows, num_experts, n * T::kBytes, k * T::kBytes)) return (int32_t)hipErrorInvalidValue;
    if (n * T::kBytes < 16 || k * T::kBytes < 16) {
      const NarrowArgs a = {static_cast<const char*>(grad_y), static_cast<const char*>(x), offsets,
                            static_cast<char*>(grad_weight), rows, 1, n, 1, k, 0, n, k, 0, (int)num_experts};
      narrow_weights<C><<<narrow_grid(num_experts * n * k), 256, 0, st>>>(a);
      return launch_status();
    }
    return whole_vectors(grad_y, x, n, k, T::kBytes)
               ? run_weights_by_size<T, C, true>(grad_y, x, offsets, grad_weight, rows, num_experts, n, k, st)
               : run_weights_by_size<T, C, false>(grad_y, x, offsets, grad_weight, rows, num_experts, n, k, st);
  });
}

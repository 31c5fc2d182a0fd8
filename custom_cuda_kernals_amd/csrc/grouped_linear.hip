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
#include "tile_product.hpp"

namespace cck {
namespace {

template <class T, class C, class P, class Q, int WP, int WQ, int FP, int FQ, bool DIRECT>
__global__ __launch_bounds__(WP* WQ * 64, DIRECT ? 2 : 1) void grouped_weights(const char* __restrict__ grad,
                                                              const char* __restrict__ x,
                                                              const int64_t* __restrict__ offsets,
                                                              char* __restrict__ out, int64_t rows, int n, int k,
                                                              int tiles_p, int tiles_q) {
  using Prod = Product<T, P, Q, NoScales, NoScales, WP, WQ, FP, FQ, DIRECT>;
  constexpr int BP = WP * FP * 16, BQ = WQ * FQ * 16;
  __shared__ __attribute__((aligned(1024))) char lds0[Prod::kStage];
  __shared__ __attribute__((aligned(1024))) char lds1[Prod::kStage];

  const int each = tiles_p * tiles_q;
  const int t = xcd_contiguous(blockIdx.x, gridDim.x), e = t / each;
  int tp, tq;
  tile_order(t - e * each, tiles_p, tiles_q, &tp, &tq);
  const int64_t lo = clamp_row(offsets[e], rows), hi = clamp_row(offsets[e + 1], rows);
  const int64_t length = hi > lo ? hi - lo : 0;
  const int p0 = tp * BP, q0 = tq * BQ;
  const int height = n - p0 < BP ? n - p0 : BP, width = k - q0 < BQ ? k - q0 : BQ;
  P p(grad + (lo * n + p0) * T::kBytes, (int64_t)n * T::kBytes, height, length);
  Q q(x + (lo * k + q0) * T::kBytes, (int64_t)k * T::kBytes, width, length);
  f32x4 acc[FP][FQ] = {};
  constexpr int kDepth = kRowBytes / T::kBytes;
  Prod::run(p, q, NoScales(), NoScales(), (int)((length + kDepth - 1) / kDepth), (LdsPtr)lds0, (LdsPtr)lds1, acc);

  const int wave = threadIdx.x >> 6;
  const bool aligned = k % C::VEC == 0 && aligned16(out);
  store_tile<C, false>(acc, out + (((int64_t)e * n + p0) * k + q0) * T::kBytes, k,
                                       (wave / WQ) * FP * 16, (wave % WQ) * FQ * 16, height, width, aligned);
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
    if (rows <= 0 || length <= 0 || cols <= 0) return (int32_t)hipSuccess;
    if (!sizes_ok(rows, groups, cols * T::kBytes, length * T::kBytes)) return (int32_t)hipErrorInvalidValue;
    const RowsArgs a = {static_cast<const char*>(x), static_cast<const char*>(w), nullptr, nullptr, offsets,
                        static_cast<char*>(out), rows, length, (int)groups, (int)cols, 0, 0};
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (whole_vectors(x, w, cols, length, T::kBytes)) return launch_rows<T, C, QROWS, 2, 2, 4, 4, true>(a, st);
    return launch_rows<T, C, QROWS, 2, 2, 4, 4, false>(a, st);
  });
}

template <class T, class C, int WP, int WQ, int FP, int FQ, bool DIRECT>
int32_t run_weights(const void* grad, const void* x, const int64_t* offsets, void* out, int64_t rows, int64_t groups,
                    int64_t n, int64_t k, hipStream_t st) {
  constexpr int BP = WP * FP * 16, BQ = WQ * FQ * 16, NW = WP * WQ;
  const int64_t tiles_p = (n + BP - 1) / BP, tiles_q = (k + BQ - 1) / BQ;
  if (groups * tiles_p * tiles_q * NW * 64 >= kMaxThreads) return (int32_t)hipErrorInvalidValue;
  grouped_weights<T, C, ColOperand<T, BP, NW>, ColOperand<T, BQ, NW>, WP, WQ, FP, FQ, DIRECT>
      <<<(unsigned)(groups * tiles_p * tiles_q), NW * 64, 0, st>>>(
          static_cast<const char*>(grad), static_cast<const char*>(x), offsets, static_cast<char*>(out), rows, (int)n,
          (int)k, (int)tiles_p, (int)tiles_q);
  return launch_status();
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
    if (whole_vectors(grad_y, x, n, k, T::kBytes)) {
      return run_weights<T, C, 2, 2, 4, 4, true>(grad_y, x, offsets, grad_weight, rows, num_experts, n, k, st);
    }
    return run_weights<T, C, 2, 2, 4, 4, false>(grad_y, x, offsets, grad_weight, rows, num_experts, n, k, st);
  });
}

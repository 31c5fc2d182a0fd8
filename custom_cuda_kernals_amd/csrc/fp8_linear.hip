// Products of FP8 codes with a scale for each block of 128 (block_product.hpp), and the
// quantiser of their activations: one scale for 128 neighbours of a row, so that a row's
// codes do not depend on its neighbours, as those of 128 x 128 tiles do.
//
//   scale = max(amax / FP8_MAX, 1e-12)    code = fp8(x / scale)
//
// bit for bit as the other granularities. The quantiser is bound by HBM: 8192 x 4096 bf16,
// 102 MB, 20 us, 5.1 TB/s; the sixteen lanes of a group meet by lane permutations, without LDS.
#include "block_product.hpp"

namespace cck {
namespace {

constexpr int kGroup = 128, kLanes = 16, kEach = kGroup / kLanes;  // elements; lanes that share them; of a lane

template <class C>
struct AmaxOf {
  using type = std::conditional_t<C::kBytes == 4, MaxU32, MaxPkU16>;
};

// A lane has eight neighbours of a row, sixteen lanes a group. WHOLE: rows are whole groups and
// aligned, so x is one run of them.
template <class C, int FMT, bool WHOLE>
__global__ __launch_bounds__(256) void fp8_group_quant(const char* __restrict__ x, uint8_t* __restrict__ codes,
                                                       float* __restrict__ scales, int64_t groups, int of_row,
                                                       int64_t width) {
  constexpr int kVectors = kEach / C::VEC;
  // Every lane of a wave takes part in its group's maximum: those past the end on the last group.
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) / kLanes; i - (threadIdx.x & 63) / kLanes < groups;
       i += (int64_t)gridDim.x * (256 / kLanes)) {
    const bool live = i < groups;
    const int64_t group = live ? i : groups - 1;
    const int at = (int)(threadIdx.x & (kLanes - 1)) * kEach;
    int64_t first;
    int count = kEach;
    if constexpr (WHOLE) {
      first = group * kGroup + at;
    } else {
      const int64_t row = group / of_row, col = (group - row * of_row) * kGroup + at;
      first = row * width + col;
      count = width - col < kEach ? (int)(width - col) : kEach;
    }
    u32x4 w[kVectors];
    if (WHOLE || count == kEach) {
#pragma unroll
      for (int v = 0; v < kVectors; ++v) {
        w[v] = WHOLE ? ld_stream(reinterpret_cast<const u32x4*>(x + first * C::kBytes) + v)
                     : *reinterpret_cast<const u32x4_any*>(x + first * C::kBytes + v * 16);
      }
    } else {
#pragma unroll
      for (int v = 0; v < kVectors; ++v) {
        float f[C::VEC];
#pragma unroll
        for (int j = 0; j < C::VEC; ++j) f[j] = v * C::VEC + j < count ? C::load1(x, first + v * C::VEC + j) : 0.0f;
        w[v] = C::pack(f);
      }
    }
    uint32_t acc = 0;
    const typename AmaxOf<C>::type most;
#pragma unroll
    for (int v = 0; v < kVectors; ++v) acc = C::absmax_vec(w[v], acc);
    acc = most(acc, dpp<kDppQuadXor1>(acc));
    acc = most(acc, dpp<kDppQuadXor2>(acc));
    acc = most(acc, dpp<kDppRowHalfMirror>(acc));
    acc = most(acc, dpp<kDppRowMirror>(acc));
    const float amax = C::absmax_to_float(acc);
    const float s = scale_from_amax<FMT>(amax), r = 1.0f / s;
    float f[kEach];
#pragma unroll
    for (int v = 0; v < kVectors; ++v) {
      float g[C::VEC];
      C::unpack(w[v], g);
#pragma unroll
      for (int j = 0; j < C::VEC; ++j) f[v * C::VEC + j] = g[j];
    }
    uint32_t out[kEach / 4];
    if (fast_path_ok<FMT>(s, r, amax)) {
      quant_fast<FMT, kEach>(f, s, r, out);
    } else {
      quant_exact<FMT, kEach>(f, s, out);
    }
    if (!live || count <= 0) continue;
    if ((threadIdx.x & (kLanes - 1)) == 0) scales[group] = s;
    if (WHOLE) {
      *reinterpret_cast<u32x2*>(codes + first) = (u32x2){out[0], out[1]};
    } else if (count == kEach) {
      *reinterpret_cast<u32x2_any*>(codes + first) = (u32x2){out[0], out[1]};
    } else {
      store_codes_partial<kEach>(out, count, codes + first);
    }
  }
}

template <class C, int FMT>
int32_t run_group_quant(const void* x, uint8_t* codes, float* scale, int64_t rows, int64_t width, hipStream_t st) {
  const int64_t of_row = (width + kGroup - 1) / kGroup, groups = rows * of_row;
  const unsigned grid = flat_grid(groups * kLanes, 256, int64_t(1) << 20);
  const char* from = static_cast<const char*>(x);
  if (width % kGroup == 0 && host_aligned(x, 16) && host_aligned(codes, 8)) {
    fp8_group_quant<C, FMT, true><<<grid, 256, 0, st>>>(from, codes, scale, groups, (int)of_row, width);
  } else {
    fp8_group_quant<C, FMT, false><<<grid, 256, 0, st>>>(from, codes, scale, groups, (int)of_row, width);
  }
  return launch_status();
}

}  // namespace
}  // namespace cck

using namespace cck;

extern "C" int32_t launch_fp8_quant_group_fwd(const void* x, uint8_t* x_fp8, float* scale, int64_t m, int64_t n,
                                              int32_t dtype, int32_t fp8_format, void* stream) {
  return with_codec(dtype, [&](auto codec) {
    return with_fp8(fp8_format, [&](auto fmt) {
      if (m <= 0 || n <= 0) return (int32_t)hipSuccess;
      if (n > INT32_MAX || m > INT64_MAX / 64 / n) return (int32_t)hipErrorInvalidValue;
      return run_group_quant<decltype(codec), decltype(fmt)::value>(x, x_fp8, scale, m, n,
                                                                    static_cast<hipStream_t>(stream));
    });
  });
}

extern "C" int32_t launch_fp8_block_linear_fwd(const void* x, const float* x_scale, const void* w, const float* w_scale,
                                               const int64_t* offsets, void* y, int64_t rows, int64_t num_experts,
                                               int64_t n, int64_t k, int32_t x_block_rows, int32_t x_format,
                                               int32_t w_format, int32_t dtype, void* stream) {
  return with_codec(dtype, [&](auto codec) {
    using C = decltype(codec);
    const auto is_fp8 = [](int32_t tag) { return tag == kF8E4M3 || tag == kF8E5M2; };
    if (!is_fp8(x_format) || !is_fp8(w_format) || (x_block_rows != 1 && x_block_rows != 128)) return (int32_t)hipErrorInvalidValue;
    if (rows <= 0 || n <= 0 || k < 0) return (int32_t)hipSuccess;
    if (!sizes_ok(rows, num_experts, n * C::kBytes, k)) return (int32_t)hipErrorInvalidValue;
    if (offsets == nullptr && num_experts != 1) return (int32_t)hipErrorInvalidValue;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (k == 0) return launch_zero_rows<C>(y, rows * n, st);
    BlockArgs a = {};
    a.rows = {static_cast<const char*>(x), static_cast<const char*>(w), nullptr, nullptr, offsets,
              static_cast<char*>(y), rows, k, (int)num_experts, (int)n, 0, 0, 0};
    a.x_scale = x_scale;
    a.w_scale = w_scale;
    a.blocks = (int)((k + 127) / 128);
    a.x_shift = x_block_rows == 128 ? 7 : 0;
    a.out_dtype = dtype;
    return with_fp8(x_format, [&](auto fx) {
      return with_fp8(w_format, [&](auto fw) {
        return launch_block_linear<decltype(fx)::value, decltype(fw)::value, C::kBytes == 4>(a, st);
      });
    });
  });
}

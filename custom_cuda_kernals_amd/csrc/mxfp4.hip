// OCP MXFP4 (microscaling formats, v1.0): 32 neighbours of a row share a power of
// two, and each is an e2m1 code (0, 0.5, 1, 1.5, 2, 3, 4 or 6, and a sign).
//
//   X     = 2^(floor(log2(max |x|)) - 2), at least 2^-127       (an E8M0 byte, bias 127)
//   code  = e2m1(x / X), to nearest, ties to the even code, beyond 6 to 6
//   value = code * X
//
// floor(log2 |x|) is the fp32 exponent field, so a block's scale byte is that of
// its largest magnitude less 2, or 0 if that is negative. A block with a NaN or an
// infinity gets the byte 255 (NaN), and zero codes. Codes are two a byte, the lower
// element in the lower half; a row's last block is filled up with zeros.
//
// Quantiser and inverse are bound by HBM: [14336, 4096] bf16 and back take 49 us (6.1 TB/s). The
// product (tile_product.hpp) takes codes and scales as they are to the scaled matrix
// instructions: 16 rows, 14336 x 4096 8.6 us, where the launch's ramp is half; 8192 rows on
// 8 experts 316 us, 3.0 PFLOP/s, of tiles whose ends cost as much as ten of their 16 steps.
#include "tile_product.hpp"

namespace cck {
namespace {

constexpr int kBlock = 32;    // elements of a scale
constexpr int kQuarter = 8;   // elements of a thread: four threads share a block
constexpr int kThreads = 256;

// The first `bytes` (below 16) at p, zeros after them. BYTES: of an element.
template <int BYTES>
__device__ inline u32x4 load_short(const char* p, int bytes) {
  u32x4 v = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int i = 0; i < 16 / BYTES; ++i) {
    if (i * BYTES < bytes) {
      uint32_t e;
      if constexpr (BYTES == 4) e = *reinterpret_cast<const u32_any*>(p + i * 4);
      if constexpr (BYTES == 2) e = *reinterpret_cast<const u16_any*>(p + i * 2);
      v[i * BYTES / 4] |= e << (8 * (i * BYTES % 4));
    }
  }
  return v;
}

// Eight elements from element `first` of x, of which `count` (0 .. 8) exist; zeros after them.
template <class C, bool WHOLE>
__device__ inline void load_quarter(const void* x, int64_t first, int count, float (&f)[kQuarter]) {
  const char* p = static_cast<const char*>(x) + first * C::kBytes;
#pragma unroll
  for (int v = 0; v < kQuarter / C::VEC; ++v) {
    u32x4 w;
    if constexpr (WHOLE) {
      w = ld_stream(reinterpret_cast<const u32x4*>(p) + v);
    } else {
      const int part = (count - v * C::VEC) * C::kBytes;
      w = part >= 16 ? *reinterpret_cast<const u32x4_any*>(p + v * 16) : load_short<C::kBytes>(p + v * 16, part);
    }
    float g[C::VEC];
    C::unpack(w, g);
#pragma unroll
    for (int i = 0; i < C::VEC; ++i) f[v * C::VEC + i] = g[i];
  }
}

// Four bytes of codes of eight values, all |v| < 8. v_cvt_scalef32_pk_fp4_f32 with
// scale 1 rounds to nearest even and saturates.
__device__ inline uint32_t encode8(const float (&v)[kQuarter]) {
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], 1.0f, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], 1.0f, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], 1.0f, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], 1.0f, 3);
}

// One thread a quarter block. FLAT: rows are whole blocks and x is aligned, so
// x is one run of blocks.
template <class C, bool FLAT>
__global__ __launch_bounds__(kThreads) void mxfp4_quant(const void* __restrict__ x, uint32_t* __restrict__ codes,
                                                       uint8_t* __restrict__ scales, int64_t quarters,
                                                       uint32_t row_quarters, int64_t width) {
  // The grid's last workgroup is whole too: its spare threads work on the last quarter's block, and store nothing.
  for (int64_t i0 = (int64_t)blockIdx.x * kThreads; i0 < quarters; i0 += (int64_t)gridDim.x * kThreads) {
    const int64_t i = i0 + threadIdx.x;
    const bool live = i < quarters;
    const int64_t at = live ? i : (quarters - 4) | (i & 3);
    float f[kQuarter];
    if constexpr (FLAT) {
      load_quarter<C, true>(x, at * kQuarter, kQuarter, f);
    } else {
      const int64_t row = at / row_quarters, first = (at - row * row_quarters) * kQuarter;
      const int64_t left = width - first;
      load_quarter<C, false>(x, row * width + (left > 0 ? first : 0), left < 0 ? 0 : left > 8 ? 8 : (int)left, f);
    }
    uint32_t amax = 0;
#pragma unroll
    for (int j = 0; j < kQuarter; ++j) amax = max(amax, f32_bits(f[j]) & 0x7fffffffu);
    amax = max(amax, dpp<kDppQuadXor1>(amax));
    amax = max(amax, dpp<kDppQuadXor2>(amax));
    const uint32_t exponent = amax >> 23;
    const bool finite = exponent != 255u;
    const uint32_t byte = finite ? (exponent > 2u ? exponent - 2u : 0u) : 255u;
    // 2^(127 - byte), exact: byte <= 252 where it is used.
    const float inverse = bits_f32((254u - (finite ? byte : 127u)) << 23);
#pragma unroll
    for (int j = 0; j < kQuarter; ++j) f[j] *= inverse;
    const uint32_t w = finite ? encode8(f) : 0u;
    if (live) {
      codes[i] = w;
      if ((i & 3) == 0) scales[i >> 2] = (uint8_t)byte;
    }
  }
}

// 2^(byte - 127); NaN for 255.
__device__ inline float e8m0(uint32_t byte) {
  return bits_f32(byte == 255u ? 0x7fc00000u : byte == 0u ? 0x00400000u : byte << 23);
}

__device__ inline void decode8(uint32_t w, float scale, float (&f)[kQuarter]) {
  const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0);
  const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1);
  const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2);
  const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3);
  const float v[kQuarter] = {a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
#pragma unroll
  for (int j = 0; j < kQuarter; ++j) f[j] = v[j] * scale;
}

template <class C, bool FLAT>
__global__ __launch_bounds__(kThreads) void mxfp4_dequant(const uint8_t* __restrict__ codes,
                                                         const uint8_t* __restrict__ scales, char* __restrict__ out,
                                                         int64_t quarters, uint32_t row_quarters, int64_t width) {
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < quarters; i += (int64_t)gridDim.x * kThreads) {
    float f[kQuarter];
    decode8(*reinterpret_cast<const u32_any*>(codes + i * 4), e8m0(scales[i >> 2]), f);
    if constexpr (FLAT) {
#pragma unroll
      for (int v = 0; v < kQuarter / C::VEC; ++v) {
        float part[C::VEC];
#pragma unroll
        for (int j = 0; j < C::VEC; ++j) part[j] = f[v * C::VEC + j];
        st_stream(C::pack(part), reinterpret_cast<u32x4*>(out + i * kQuarter * C::kBytes) + v);
      }
    } else {
      const int64_t row = i / row_quarters, first = (i - row * row_quarters) * kQuarter;
#pragma unroll
      for (int j = 0; j < kQuarter; ++j) {
        if (first + j < width) C::store1(out, row * width + first + j, f[j]);
      }
    }
  }
}

inline int64_t blocks_of(int64_t width) { return (width + kBlock - 1) / kBlock; }

// Rows of at most 2^31 - 1 elements (32-bit quarters), and int64 elements in all.
inline bool row_sizes_ok(int64_t rows, int64_t width) { return width <= INT32_MAX && rows <= INT64_MAX / 64 / width; }

constexpr int64_t kMaxBlocks = int64_t(1) << 20;  // workgroups; beyond it they loop

}  // namespace
}  // namespace cck

using namespace cck;

extern "C" int32_t launch_mxfp4_quant_fwd(const void* x, uint8_t* codes, uint8_t* scales, int64_t rows, int64_t width,
                                          int32_t dtype, void* stream) {
  return with_codec(dtype, [&](auto codec) {
    using C = decltype(codec);
    if (rows <= 0 || width <= 0) return (int32_t)hipSuccess;
    if (!row_sizes_ok(rows, width)) return (int32_t)hipErrorInvalidValue;
    if (!host_aligned(codes, 4)) return (int32_t)hipErrorInvalidValue;
    const int64_t row_quarters = blocks_of(width) * 4, quarters = rows * row_quarters;
    const unsigned grid = flat_grid(quarters, kThreads, kMaxBlocks);
    uint32_t* const words = reinterpret_cast<uint32_t*>(codes);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (width % kBlock == 0 && host_aligned(x, 16)) {
      mxfp4_quant<C, true><<<grid, kThreads, 0, st>>>(x, words, scales, quarters, (uint32_t)row_quarters, width);
    } else {
      mxfp4_quant<C, false><<<grid, kThreads, 0, st>>>(x, words, scales, quarters, (uint32_t)row_quarters, width);
    }
    return launch_status();
  });
}

extern "C" int32_t launch_mxfp4_dequant_fwd(const void* codes, const void* scales, void* out, int64_t rows,
                                            int64_t width, int32_t dtype, void* stream) {
  return with_codec(dtype, [&](auto codec) {
    using C = decltype(codec);
    if (rows <= 0 || width <= 0) return (int32_t)hipSuccess;
    if (!row_sizes_ok(rows, width)) return (int32_t)hipErrorInvalidValue;
    const int64_t row_quarters = blocks_of(width) * 4, quarters = rows * row_quarters;
    const unsigned grid = flat_grid(quarters, kThreads, kMaxBlocks);
    const uint8_t *c = static_cast<const uint8_t*>(codes), *e = static_cast<const uint8_t*>(scales);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (width % kBlock == 0 && host_aligned(out, 16)) {
      mxfp4_dequant<C, true><<<grid, kThreads, 0, st>>>(c, e, static_cast<char*>(out), quarters,
                                                        (uint32_t)row_quarters, width);
    } else {
      mxfp4_dequant<C, false><<<grid, kThreads, 0, st>>>(c, e, static_cast<char*>(out), quarters,
                                                         (uint32_t)row_quarters, width);
    }
    return launch_status();
  });
}

extern "C" int32_t launch_mxfp4_linear_fwd(const void* x_codes, const void* x_scales, const void* w_codes,
                                           const void* w_scales, const int64_t* offsets, void* y, int64_t rows,
                                           int64_t num_experts, int64_t n, int64_t blocks, int32_t dtype,
                                           void* stream) {
  return with_codec(dtype, [&](auto codec) {
    using C = decltype(codec);
    if (rows <= 0 || n <= 0 || blocks < 0) return (int32_t)hipSuccess;
    if (!sizes_ok(rows, num_experts, n * C::kBytes, blocks * 16)) return (int32_t)hipErrorInvalidValue;
    if (offsets == nullptr && num_experts != 1) return (int32_t)hipErrorInvalidValue;
    if (blocks == 0) return launch_zero_rows<C>(y, rows * n, static_cast<hipStream_t>(stream));
    const RowsArgs a = {static_cast<const char*>(x_codes), static_cast<const char*>(w_codes),
                        static_cast<const char*>(x_scales), static_cast<const char*>(w_scales), offsets,
                        static_cast<char*>(y), rows, blocks * 16, (int)num_experts, (int)n, 0, 0, 0};
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const bool whole = blocks % 4 == 0 && host_aligned(x_codes, 16) && host_aligned(w_codes, 16) &&
                       host_aligned(x_scales, 4) && host_aligned(w_scales, 4);
    return whole ? launch_rows_by_size<ElemFP4, C, true>(a, st) : launch_rows_by_size<ElemFP4, C, false>(a, st);
  });
}

// Rotary positions: each pair (a, b) of a head's elements is turned by the angle
// position * frequency[i] of its pair i,
//
//   a' = factor (a cos - b sin)     b' = factor (b cos + a sin)
//
// with pairs (x[i], x[i + R / 2]) or (x[2 i], x[2 i + 1]) of the first R elements; the
// others stay. The inverse turns by the negative angle, which is the gradient too: with
// factor s the rotation is s times an orthogonal map. launch_rope_at_fwd writes q and k;
// launch_rope_to_cache_fwd writes q, and k and v to slots of a paged cache.
//
// Bound by HBM, q and k once each way. The angles are not read but made: a workgroup has a
// few tokens, and each of its threads the sine and cosine of one (token, pair), into LDS,
// while its first vectors are on their way. The angle is formed in float64, where whole
// turns come off exactly: position 10^6 keeps the last bits that float32 angles lose from
// some hundred positions on.
#include "launch.hpp"

namespace cck {
namespace {

constexpr int kThreads = 256;
constexpr int kInFlight = 4;        // items of a thread whose loads are issued together
constexpr int kMaxHalf = 1024;      // pairs of a head

// sin and cos of position * frequency. In quarter turns the whole part picks the quadrant
// and the rest, at most half a quarter turn, is exact in float64; its float32 rounding is
// 2^-25 of a radian. The series of Taylor to x^9 and x^10 end below 2e-9 at pi / 4.
__device__ inline f32x2 sin_cos(double position, double frequency) {
  const double quarters = position * (frequency * 0.63661977236758134308);  // 2 / pi
  const double whole = __builtin_rint(quarters);
  const float x = (float)((quarters - whole) * 1.57079632679489661923);
  const int quadrant = (int)(whole - 4.0 * __builtin_floor(whole * 0.25));
  const float y = x * x;
  float s = __builtin_fmaf(y, 1.0f / 362880.0f, -1.0f / 5040.0f);
  s = __builtin_fmaf(y, s, 1.0f / 120.0f);
  s = __builtin_fmaf(y, s, -1.0f / 6.0f);
  s = __builtin_fmaf(y * x, s, x);
  float c = __builtin_fmaf(y, -1.0f / 3628800.0f, 1.0f / 40320.0f);
  c = __builtin_fmaf(y, c, -1.0f / 720.0f);
  c = __builtin_fmaf(y, c, 1.0f / 24.0f);
  c = __builtin_fmaf(y, c, -0.5f);
  c = __builtin_fmaf(y, c, 1.0f);
  const float a = quadrant & 1 ? c : s, b = quadrant & 1 ? s : c;
  return (f32x2){quadrant & 2 ? -a : a, (quadrant + 1) & 2 ? -b : b};
}

// A tensor of heads: element strides of a token and of a head.
struct Heads {
  const char* from;
  char* to;
  int64_t from_token, from_head, to_token, to_head;
  int heads;
};

struct Args {
  Heads q, k, v;  // k.to and v.to: the caches, for which to_token is a slot's stride
  const int64_t *positions, *slots;
  const double* frequencies;
  int64_t tokens, slot_count;
  int dim, half, block_tokens, slices;
  float factor, sine_sign, key_scale, key_inverse, value_scale, value_inverse;
};

// What a head's D elements are cut into, in this order: vectors of whole pairs, single
// pairs, and for what is copied vectors and single elements.
struct Pieces {
  int turn_vectors, turn_pairs, copy_vectors, copies;
  __host__ __device__ int all() const { return turn_vectors + turn_pairs + copy_vectors + copies; }
};
template <class C, bool INTERLEAVED>
__host__ __device__ inline Pieces pieces_of(int dim, int half, bool copy) {
  constexpr int kPairs = INTERLEAVED ? C::VEC / 2 : C::VEC;  // of a vector
  const int rest = copy ? dim - 2 * half : 0;
  return {half / kPairs, half % kPairs, rest / C::VEC, rest % C::VEC};
}

// Where results go: elements of C, or FP8 codes of a cache. NT: past the caches.
template <class C, bool NT>
struct Plain {
  static constexpr int kBytes = C::kBytes;
  __device__ static void vector(const float (&f)[C::VEC], char* p, float, float) {
    const u32x4 w = C::pack(f);
    if constexpr (NT) {
      __builtin_nontemporal_store(w, reinterpret_cast<u32x4_any*>(p));
    } else {
      *reinterpret_cast<u32x4_any*>(p) = w;
    }
  }
  __device__ static void one(float f, char* p, float, float) { C::store1(p, 0, f); }
};

// x / scale to the nearest code, beyond the largest value to it; NaN stays NaN.
template <class C, int FMT>
struct Codes {
  static constexpr int kBytes = 1;
  __device__ static float limit(float x, float most) { return x > most ? most : x < -most ? -most : x; }
  __device__ static float quotient(float x, float scale, float inverse) {
    const float most = Fp8<FMT>::kMax;
    return limit(div_by_scale(limit(x, 2.0f * most * scale), scale, inverse), most);
  }
  __device__ static void vector(const float (&f)[C::VEC], char* p, float scale, float inverse) {
    uint32_t w[C::VEC / 4];
#pragma unroll
    for (int i = 0; i < C::VEC / 4; ++i) {
      float g[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) g[j] = quotient(f[4 * i + j], scale, inverse);
      w[i] = Fp8<FMT>::cvt4(g[0], g[1], g[2], g[3]);
    }
    if constexpr (C::VEC == 8) {
      *reinterpret_cast<u32x2_any*>(p) = (u32x2){w[0], w[C::VEC / 4 - 1]};
    } else {
      *reinterpret_cast<u32_any*>(p) = w[0];
    }
  }
  __device__ static void one(float f, char* p, float scale, float inverse) {
    const float g = quotient(f, scale, inverse);
    *reinterpret_cast<uint8_t*>(p) = (uint8_t)Fp8<FMT>::cvt4(g, g, g, g);
  }
};

enum Kind { kNone, kTurnVector, kTurnPair, kCopyVector, kCopy };

// One piece of one head of one token.
template <class C, bool INTERLEAVED>
struct Item {
  static constexpr int kPairs = INTERLEAVED ? C::VEC / 2 : C::VEC;
  int kind, target, first;  // target: 0 q, 1 k, 2 v; first: its first pair, or its first element if copied
  uint32_t table;           // of its token
  char* to;
  u32x4 w[INTERLEAVED ? 1 : 2];
  float a, b;
};

template <bool NT>
__device__ inline u32x4 load16(const char* p) {
  if constexpr (NT) return __builtin_nontemporal_load(reinterpret_cast<const u32x4_any*>(p));
  return *reinterpret_cast<const u32x4_any*>(p);
}

// WHOLE: only vectors of pairs.
template <class C, class KC, bool INTERLEAVED, bool CACHE, bool WHOLE, bool NT>
__global__ __launch_bounds__(kThreads) void rope_at(Args a, int copy_q) {
  using It = Item<C, INTERLEAVED>;
  using QC = Plain<C, NT>;
  extern __shared__ f32x2 table[];  // [block_tokens][half]: sine and cosine
  const Pieces pq = pieces_of<C, INTERLEAVED>(a.dim, a.half, copy_q != 0);
  const Pieces pk = pieces_of<C, INTERLEAVED>(a.dim, a.half, CACHE || copy_q != 0);
  // WHOLE: values in pieces as keys, which are not turned.
  const int value_vectors = a.dim / C::VEC, of_value = WHOLE ? pk.all() : value_vectors + a.dim % C::VEC;
  const int of_q = pq.all() * a.q.heads, of_qk = of_q + pk.all() * a.k.heads;
  const int of_token = of_qk + (CACHE ? of_value * a.v.heads : 0);
  const int64_t groups = (a.tokens + a.block_tokens - 1) / a.block_tokens;

  for (int64_t id = blockIdx.x; id < groups * a.slices; id += gridDim.x) {
    const int64_t t0 = id / a.slices * a.block_tokens;
    const int slice = (int)(id % a.slices);
    const int count = a.tokens - t0 < a.block_tokens ? (int)(a.tokens - t0) : a.block_tokens;
    const int total = count * of_token;
    const int each = (total + a.slices - 1) / a.slices, begin = slice * each;
    const int end = begin + each < total ? begin + each : total;

    auto load = [&](int i, It& it) __attribute__((always_inline)) {
      it.kind = kNone;
      if (i >= end) return;
      const int t = i / of_token;
      int r = i - t * of_token, head, piece;
      const int64_t token = t0 + t;
      const Heads& h = r < of_q ? a.q : r < of_qk ? a.k : a.v;
      it.target = r < of_q ? 0 : r < of_qk ? 1 : 2;
      it.table = (uint32_t)(t * a.half);
      Pieces p = it.target == 0 ? pq : pk;
      if (it.target == 2) {
        r -= of_qk;
        if constexpr (!WHOLE) p = {0, 0, value_vectors, of_value - value_vectors};
      } else if (it.target == 1) {
        r -= of_q;
      }
      const int n = p.all();
      head = r / n;
      piece = r - head * n;
      const char* from = h.from + (token * h.from_token + (int64_t)head * h.from_head) * C::kBytes;
      const int bytes = CACHE && it.target > 0 ? KC::kBytes : C::kBytes;
      int64_t row = token;
      if (CACHE && it.target > 0) {
        row = a.slots[token];
        if (row < 0 || row >= a.slot_count) return;  // a token without a slot is not written
      }
      it.to = h.to + (row * h.to_token + (int64_t)head * h.to_head) * bytes;
      if (piece < p.turn_vectors) {
        it.kind = kTurnVector;
        it.first = piece * It::kPairs;
        const int e = INTERLEAVED ? 2 * it.first : it.first;
        it.w[0] = load16<NT>(from + e * C::kBytes);
        if constexpr (!INTERLEAVED) it.w[1] = load16<NT>(from + (e + a.half) * C::kBytes);
        it.to += (int64_t)e * bytes;
        return;
      }
      if constexpr (!WHOLE) {
        piece -= p.turn_vectors;
        if (piece < p.turn_pairs) {
          it.kind = kTurnPair;
          it.first = p.turn_vectors * It::kPairs + piece;
          const int e = INTERLEAVED ? 2 * it.first : it.first;
          it.a = C::load1(from, e);
          it.b = C::load1(from, e + (INTERLEAVED ? 1 : a.half));
          it.to += (int64_t)e * bytes;
          return;
        }
        piece -= p.turn_pairs;
        const int base = it.target == 2 ? 0 : 2 * a.half;
        it.kind = piece < p.copy_vectors ? kCopyVector : kCopy;
        const int e = base + (piece < p.copy_vectors ? piece * C::VEC
                                                     : p.copy_vectors * C::VEC + piece - p.copy_vectors);
        if (it.kind == kCopyVector) {
          it.w[0] = load16<NT>(from + (int64_t)e * C::kBytes);
        } else {
          it.a = C::load1(from, e);
        }
        it.to += (int64_t)e * bytes;
      }
    };

    auto turn = [&](float& x, float& y, const f32x2& sc) {
      const float u = __builtin_fmaf(x, sc[1], -(y * sc[0])), v = __builtin_fmaf(y, sc[1], x * sc[0]);
      x = u;
      y = v;
    };
    // fn(scale, inverse, codec) of the item's target.
    auto store = [&](const It& it) __attribute__((always_inline)) {
      if (it.kind == kNone) return;
      constexpr bool kCodes = CACHE && KC::kBytes != C::kBytes;
      const bool cached = kCodes && it.target > 0;
      const float scale = it.target == 2 ? a.value_scale : a.key_scale;
      const float inverse = it.target == 2 ? a.value_inverse : a.key_inverse;
      const f32x2* sc = table + it.table + it.first;
      float f[C::VEC];
      C::unpack(it.w[0], f);
      if (it.kind == kTurnVector) {
        if constexpr (INTERLEAVED) {
#pragma unroll
          for (int i = 0; i < It::kPairs; ++i) {
            if (!WHOLE || !CACHE || it.target < 2) turn(f[2 * i], f[2 * i + 1], sc[i]);
          }
        } else {
          float g[C::VEC];
          C::unpack(it.w[1], g);
#pragma unroll
          for (int i = 0; i < C::VEC; ++i) {
            if (!WHOLE || !CACHE || it.target < 2) turn(f[i], g[i], sc[i]);
          }
          if (cached) {
            KC::vector(g, it.to + (int64_t)a.half * KC::kBytes, scale, inverse);
          } else {
            QC::vector(g, it.to + (int64_t)a.half * C::kBytes, 0.0f, 0.0f);
          }
        }
        if (cached) {
          KC::vector(f, it.to, scale, inverse);
        } else {
          QC::vector(f, it.to, 0.0f, 0.0f);
        }
        return;
      }
      if constexpr (!WHOLE) {
        if (it.kind == kCopyVector) {
          if (cached) {
            KC::vector(f, it.to, scale, inverse);
          } else {
            QC::vector(f, it.to, 0.0f, 0.0f);
          }
          return;
        }
        float x = it.a, y = it.b;
        const bool pair = it.kind == kTurnPair;
        if (pair) turn(x, y, *sc);
        const int64_t apart = INTERLEAVED ? 1 : a.half;
        if (cached) {
          KC::one(x, it.to, scale, inverse);
          if (pair) KC::one(y, it.to + apart * KC::kBytes, scale, inverse);
        } else {
          C::store1(it.to, 0, x);
          if (pair) C::store1(it.to, apart, y);
        }
      }
    };

    It items[kInFlight];
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) load(begin + (int)threadIdx.x + u * kThreads, items[u]);
    for (int i = threadIdx.x; i < count * a.half; i += kThreads) {
      const int t = i / a.half;
      const f32x2 sc = sin_cos((double)a.positions[t0 + t], a.frequencies[i - t * a.half]);
      table[i] = (f32x2){sc[0] * a.sine_sign, sc[1] * a.factor};
    }
    __syncthreads();
    for (int i = begin + (int)threadIdx.x;;) {
#pragma unroll
      for (int u = 0; u < kInFlight; ++u) store(items[u]);
      i += kInFlight * kThreads;
      if (i - (int)threadIdx.x >= end) break;
#pragma unroll
      for (int u = 0; u < kInFlight; ++u) load(i + u * kThreads, items[u]);
    }
    __syncthreads();  // the table is read
  }
}

// Tokens a workgroup takes and workgroups a token's items are spread over.
template <class C, class KC, bool INTERLEAVED, bool CACHE, bool WHOLE, bool NT>
int32_t run(Args a, bool copy_q, int of_token, hipStream_t st) {
  const int64_t room = a.half > 0 ? kThreads / a.half : 8;
  int64_t each = a.tokens / 1024;
  each = each < 1 ? 1 : each;
  const int64_t most = room < 1 ? 1 : room;
  a.block_tokens = (int)(each < most ? each : most);
  const int64_t groups = (a.tokens + a.block_tokens - 1) / a.block_tokens;
  a.slices = groups < 512 ? (of_token * a.block_tokens + kThreads - 1) / kThreads : 1;
  const int64_t blocks = groups * a.slices;
  const unsigned grid = (unsigned)(blocks < (int64_t(1) << 22) ? blocks : (int64_t(1) << 22));
  const size_t lds = (size_t)a.block_tokens * a.half * sizeof(f32x2);
  rope_at<C, KC, INTERLEAVED, CACHE, WHOLE, NT><<<grid, kThreads, lds, st>>>(a, copy_q ? 1 : 0);
  return launch_status();
}

template <class C, class KC, bool INTERLEAVED, bool CACHE>
int32_t by_shape(const Args& a, bool copy_q, hipStream_t st) {
  const Pieces q = pieces_of<C, INTERLEAVED>(a.dim, a.half, copy_q);
  const Pieces k = pieces_of<C, INTERLEAVED>(a.dim, a.half, CACHE || copy_q);
  const bool whole = k.turn_pairs + k.copy_vectors + k.copies == 0 && (!CACHE || a.dim % C::VEC == 0);
  const int value = whole ? k.all() : a.dim / C::VEC + a.dim % C::VEC;
  const int64_t of_token = (int64_t)q.all() * a.q.heads + (int64_t)k.all() * a.k.heads +
                           (CACHE ? (int64_t)value * a.v.heads : 0);
  // Item numbers of a workgroup's tokens are 32-bit.
  if (of_token > (int64_t(1) << 21)) return (int32_t)hipErrorInvalidValue;
  if (of_token == 0) return (int32_t)hipSuccess;
  if (!whole) return run<C, KC, INTERLEAVED, CACHE, false, false>(a, copy_q, (int)of_token, st);
  const int64_t bytes = a.tokens * (a.q.heads + a.k.heads) * a.dim * C::kBytes;
  if (bytes >= (int64_t(1) << 26)) return run<C, KC, INTERLEAVED, CACHE, true, true>(a, copy_q, (int)of_token, st);
  return run<C, KC, INTERLEAVED, CACHE, true, false>(a, copy_q, (int)of_token, st);
}

bool sizes_ok(const Args& a) {
  return a.dim >= 1 && a.dim <= 2 * kMaxHalf && a.half >= 0 && 2 * a.half <= a.dim && a.q.heads >= 0 && a.k.heads >= 0;
}

}  // namespace
}  // namespace cck

using namespace cck;

extern "C" int32_t launch_rope_at_fwd(const void* q, const void* k, void* q_out, void* k_out, const int64_t* positions,
                                      const void* frequencies, const int64_t* strides, int64_t tokens,
                                      int64_t n_q_heads, int64_t n_kv_heads, int64_t head_dim, int64_t half,
                                      int32_t interleaved, int32_t inverse, float factor, int32_t dtype, void* stream) {
  return with_codec(dtype, [&](auto codec) {
    using C = decltype(codec);
    if (tokens <= 0 || head_dim <= 0) return (int32_t)hipSuccess;
    if (n_q_heads > INT32_MAX || n_kv_heads > INT32_MAX || head_dim > 2 * kMaxHalf || half > kMaxHalf) {
      return (int32_t)hipErrorInvalidValue;
    }
    Args a = {};
    a.q = {(const char*)q, (char*)q_out, strides[0], strides[1], strides[4], strides[5], (int)n_q_heads};
    a.k = {(const char*)k, (char*)k_out, strides[2], strides[3], strides[6], strides[7], (int)n_kv_heads};
    a.positions = positions;
    a.frequencies = (const double*)frequencies;
    a.tokens = tokens;
    a.dim = (int)head_dim;
    a.half = (int)half;
    a.factor = factor;
    a.sine_sign = inverse ? -factor : factor;
    if (!sizes_ok(a)) return (int32_t)hipErrorInvalidValue;
    const bool copy = !(q == q_out && k == k_out);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    return interleaved ? by_shape<C, Plain<C, false>, true, false>(a, copy, st)
                       : by_shape<C, Plain<C, false>, false, false>(a, copy, st);
  });
}

extern "C" int32_t launch_rope_to_cache_fwd(const void* q, const void* k, const void* v, void* q_out, void* key_cache,
                                            void* value_cache, const int64_t* slots, const int64_t* positions,
                                            const void* frequencies, const int64_t* strides, int64_t tokens,
                                            int64_t n_q_heads, int64_t n_kv_heads, int64_t head_dim, int64_t half,
                                            int64_t cache_slots, int32_t interleaved, float factor, float key_scale,
                                            float value_scale, int32_t dtype, int32_t cache_dtype, void* stream) {
  return with_codec(dtype, [&](auto codec) {
    using C = decltype(codec);
    if (cache_dtype != dtype && cache_dtype != kF8E4M3 && cache_dtype != kF8E5M2) return (int32_t)hipErrorInvalidValue;
    if (tokens <= 0 || head_dim <= 0) return (int32_t)hipSuccess;
    if (n_q_heads > INT32_MAX || n_kv_heads > INT32_MAX || head_dim > 2 * kMaxHalf || half > kMaxHalf) {
      return (int32_t)hipErrorInvalidValue;
    }
    if (!(key_scale >= 1e-30f && key_scale <= 1e30f && value_scale >= 1e-30f && value_scale <= 1e30f)) {
      return (int32_t)hipErrorInvalidValue;
    }
    Args a = {};
    a.q = {(const char*)q, (char*)q_out, strides[0], strides[1], strides[6], strides[7], (int)n_q_heads};
    a.k = {(const char*)k, (char*)key_cache, strides[2], strides[3], n_kv_heads * head_dim, head_dim, (int)n_kv_heads};
    a.v = {(const char*)v, (char*)value_cache, strides[4], strides[5], n_kv_heads * head_dim, head_dim,
           (int)n_kv_heads};
    a.positions = positions;
    a.slots = slots;
    a.frequencies = (const double*)frequencies;
    a.tokens = tokens;
    a.slot_count = cache_slots;
    a.dim = (int)head_dim;
    a.half = (int)half;
    a.factor = factor;
    a.sine_sign = factor;
    a.key_scale = key_scale;
    a.key_inverse = 1.0f / key_scale;
    a.value_scale = value_scale;
    a.value_inverse = 1.0f / value_scale;
    if (!sizes_ok(a)) return (int32_t)hipErrorInvalidValue;
    const bool copy = q != q_out;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    auto run_to = [&](auto target) {
      using KC = decltype(target);
      return interleaved ? by_shape<C, KC, true, true>(a, copy, st) : by_shape<C, KC, false, true>(a, copy, st);
    };
    if (cache_dtype == kF8E4M3) return run_to(Codes<C, kF8E4M3>{});
    if (cache_dtype == kF8E5M2) return run_to(Codes<C, kF8E5M2>{});
    return run_to(Plain<C, false>{});
  });
}

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
// Bound by HBM, q and k once each way. The angles are not read but made: each thread of a
// workgroup the sine and cosine of a (token, pair), into LDS, while its vectors are on
// their way. The angle is formed in float64, where whole
// turns come off exactly: position 10^6 keeps the last bits that float32 angles lose from
// some hundred positions on.
//
// bf16, 32 + 8 heads of 128: 32768 tokens, 671 MB, 105 to 109 us, 6.2 TB/s (a copy reaches
// 5.2); 8192 tokens to a bf16 cache, 201 MB, 39 to 41 us; a decode step's 16 tokens 2.7 us.
#include "launch.hpp"

namespace cck {
namespace {

constexpr int kMaxThreads = 1024, kFewThreads = 128;
constexpr int64_t kMaxGroups = int64_t(1) << 21;  // workgroups; beyond it they loop
constexpr int kMaxHalf = 1024;                    // pairs of a head

// The workgroup's LDS writes are there for all; loads that are on their way stay so, unlike at __syncthreads.
__device__ inline void lds_written() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// sin and cos of position * frequency. In quarter turns the whole part picks the quadrant
// and the rest, at most half a quarter turn, is exact in float64; its float32 rounding is
// 2^-25 of a radian. The series of Taylor to x^9 and x^10 end below 2e-9 at pi / 4. Three float64
// roundings of the angle come before: 2^-51 of it together, which is less than the rest up to 2^28.
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
  int dim, half;
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

// Where results go: elements of C, or FP8 codes of a cache.
template <class C>
struct Plain {
  static constexpr int kBytes = C::kBytes;
  __device__ static void vector(const float (&f)[C::VEC], char* p, float, float) {
    *reinterpret_cast<u32x4_any*>(p) = C::pack(f);
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

template <bool NT>
__device__ inline u32x4 load16(const char* p) {
  if constexpr (NT) return __builtin_nontemporal_load(reinterpret_cast<const u32x4_any*>(p));
  return *reinterpret_cast<const u32x4_any*>(p);
}

// A workgroup has TOKENS tokens, and a thread the same pieces of each: where they are is
// found once, and the loads of all tokens go out together. blockIdx.y: which of a token's
// pieces, where tokens are few.
// WHOLE: only vectors of pairs, those of v being copied. NT: loads as of data read once, and stores that
// go on from the caches at once, by 32-bit offsets in a token.
template <class C, class KC, bool INTERLEAVED, bool CACHE, bool WHOLE, bool NT, int TOKENS>
__global__ __launch_bounds__(kMaxThreads) void rope_at(Args a, int copy_q) {
  constexpr int kPairs = INTERLEAVED ? C::VEC / 2 : C::VEC;
  constexpr bool kCodes = CACHE && KC::kBytes != C::kBytes;
  extern __shared__ f32x2 table[];  // [TOKENS][half]: sine and cosine
  const Pieces pq = pieces_of<C, INTERLEAVED>(a.dim, a.half, copy_q != 0);
  const Pieces pk = pieces_of<C, INTERLEAVED>(a.dim, a.half, CACHE || copy_q != 0);
  const int value_vectors = a.dim / C::VEC, of_value = WHOLE ? pk.all() : value_vectors + a.dim % C::VEC;
  const int of_q = pq.all() * a.q.heads, of_qk = of_q + pk.all() * a.k.heads;
  const int of_token = of_qk + (CACHE ? of_value * a.v.heads : 0);
  const int threads = (int)blockDim.x, stride = threads * (int)gridDim.y, begin = (int)blockIdx.y * threads;
  const int64_t groups = (a.tokens + TOKENS - 1) / TOKENS;
  // In registers: where one of several is taken, the compiler would put all arguments to scratch memory.
  char *const q_to = a.q.to, *const k_to = a.k.to, *const v_to = a.v.to;
  const int64_t cache_row = a.k.to_token * (kCodes ? KC::kBytes : C::kBytes);  // v's is as long
  const float key_scale = a.key_scale, key_inverse = a.key_inverse, value_scale = a.value_scale,
              value_inverse = a.value_inverse;

  for (int64_t id = blockIdx.x; id < groups; id += gridDim.x) {
    const int64_t t0 = id * TOKENS;
    const int count = a.tokens - t0 < TOKENS ? (int)(a.tokens - t0) : TOKENS;
    for (int i0 = begin; i0 < of_token; i0 += stride) {
      // The thread's piece: of q (target 0), k or v, and where in a token.
      const int i = i0 + (int)threadIdx.x;
      int kind = kNone, target = 0, first = 0;  // first: its first pair
      int64_t from = 0, to = 0;                 // bytes from the token's on
      if (i < of_token) {
        target = i < of_q ? 0 : i < of_qk ? 1 : 2;
        Pieces p = target == 0 ? pq : pk;
        if (!WHOLE && CACHE && target == 2) p = {0, 0, value_vectors, of_value - value_vectors};
        const int r = i - (target == 0 ? 0 : target == 1 ? of_q : of_qk), head = r / p.all();
        int piece = r - head * p.all(), e;
        if (piece < p.turn_vectors) {
          kind = kTurnVector;
          first = piece * kPairs;
          e = INTERLEAVED ? 2 * first : first;
        } else if (piece -= p.turn_vectors; piece < p.turn_pairs) {
          kind = kTurnPair;
          first = p.turn_vectors * kPairs + piece;
          e = INTERLEAVED ? 2 * first : first;
        } else {
          piece -= p.turn_pairs;
          kind = piece < p.copy_vectors ? kCopyVector : kCopy;
          e = (CACHE && target == 2 ? 0 : 2 * a.half) +
              (piece < p.copy_vectors ? piece * C::VEC : p.copy_vectors * C::VEC + piece - p.copy_vectors);
        }
        const int64_t from_head = target == 0 ? a.q.from_head : target == 1 ? a.k.from_head : a.v.from_head;
        const int64_t to_head = target == 0 ? a.q.to_head : target == 1 ? a.k.to_head : a.v.to_head;
        from = (head * from_head + e) * C::kBytes;
        to = (head * to_head + e) * (kCodes && target > 0 ? KC::kBytes : C::kBytes);
      }
      const char* base = target == 0 ? a.q.from : target == 1 ? a.k.from : a.v.from;
      const int64_t token = (target == 0 ? a.q.from_token : target == 1 ? a.k.from_token : a.v.from_token) * C::kBytes;
      const char* p = base + t0 * token + from;
      u32x4 w[TOKENS][INTERLEAVED ? 1 : 2];
      float x[TOKENS], y[TOKENS];
      const int apart = (INTERLEAVED ? 1 : a.half) * C::kBytes;  // from a to b of a pair
#pragma unroll
      for (int u = 0; u < TOKENS; ++u) {
        if (u < count && kind != kNone) {
          if (WHOLE || kind == kTurnVector || kind == kCopyVector) {
            w[u][0] = load16<NT>(p);
            if constexpr (!INTERLEAVED) {
              if (WHOLE || kind == kTurnVector) w[u][1] = load16<NT>(p + apart);
            }
          } else {
            x[u] = C::load1(p, 0);
            if (kind == kTurnPair) y[u] = C::load1(p + apart, 0);
          }
        }
        p += token;
      }
      if (i0 == begin) {
        for (int j = (int)threadIdx.x; j < count * a.half; j += threads) {
          const int t = j / a.half;
          const f32x2 sc = sin_cos((double)a.positions[t0 + t], a.frequencies[j - t * a.half]);
          table[j] = (f32x2){sc[0] * a.sine_sign, sc[1] * a.factor};
        }
        lds_written();
      }
#pragma unroll
      for (int u = 0; u < TOKENS; ++u) {
        if (u >= count) break;
        // Of this token: the same in all lanes.
        const int64_t t = t0 + u;
        const int64_t slot = CACHE ? a.slots[t] : t;
        const bool has_slot = !CACHE || (slot >= 0 && slot < a.slot_count);  // else k and v are not written
        char* const to_q = q_to + t * a.q.to_token * C::kBytes;
        const int64_t row = (has_slot ? slot : 0) * cache_row;
        const f32x2* const sc = table + u * a.half + first;
        auto turn = [&](float& c, float& d, const f32x2& by) __attribute__((always_inline)) {
          const float m = __builtin_fmaf(c, by[1], -(d * by[0])), n = __builtin_fmaf(d, by[1], c * by[0]);
          c = m;
          d = n;
        };
        // fn(where a token's are, whether as codes, their scale): where the lane's results go.
        auto to_target = [&](auto&& fn) __attribute__((always_inline)) {
          if (kind == kNone || (target > 0 && !has_slot)) return;
          if (target == 0) {
            fn(to_q, std::false_type{}, 1.0f, 1.0f);
          } else if (!CACHE || target == 1) {
            fn(k_to + row, std::bool_constant<kCodes>{}, key_scale, key_inverse);
          } else {
            fn(v_to + row, std::bool_constant<kCodes>{}, value_scale, value_inverse);
          }
        };
        if (WHOLE || kind == kTurnVector || kind == kCopyVector) {
          float f[C::VEC], g[C::VEC];
          C::unpack(w[u][0], f);
          const bool turned = WHOLE ? !CACHE || target < 2 : kind == kTurnVector;
          const bool both = !INTERLEAVED && (WHOLE || kind == kTurnVector);
          if constexpr (INTERLEAVED) {
            if (turned) {
#pragma unroll
              for (int j = 0; j < kPairs; ++j) turn(f[2 * j], f[2 * j + 1], sc[j]);
            }
          } else {
            C::unpack(w[u][1], g);
            if (turned) {
#pragma unroll
              for (int j = 0; j < C::VEC; ++j) turn(f[j], g[j], sc[j]);
            }
          }
          to_target([&](char* at, auto codes, float scale, float inverse) __attribute__((always_inline)) {
            if constexpr (decltype(codes)::value) {
              KC::vector(f, at + to, scale, inverse);
              if (both) KC::vector(g, at + to + a.half * KC::kBytes, scale, inverse);
            } else if constexpr (NT) {
              const RowBuf<true, kPolSC1 | kPolNT> row(at, 0x7fffffffu);
              row.st16(C::pack(f), (uint32_t)to);
              if (both) row.st16(C::pack(g), (uint32_t)to + (uint32_t)apart);
            } else {
              Plain<C>::vector(f, at + to, 0.0f, 0.0f);
              if (both) Plain<C>::vector(g, at + to + apart, 0.0f, 0.0f);
            }
          });
        } else if constexpr (!WHOLE) {
          float c = x[u], d = y[u];
          const bool pair = kind == kTurnPair;
          if (pair) turn(c, d, *sc);
          to_target([&](char* at, auto codes, float scale, float inverse) __attribute__((always_inline)) {
            if constexpr (decltype(codes)::value) {
              KC::one(c, at + to, scale, inverse);
              if (pair) KC::one(d, at + to + (INTERLEAVED ? 1 : a.half), scale, inverse);
            } else {
              C::store1(at + to, 0, c);
              if (pair) C::store1(at + to + apart, 0, d);
            }
          });
        }
      }
    }
    if (id + gridDim.x < groups) __syncthreads();  // the table is read
  }
}

template <class C, class KC, bool INTERLEAVED, bool CACHE, bool WHOLE, bool NT, int TOKENS>
int32_t run(const Args& a, bool copy_q, int of_token, hipStream_t st) {
  const int64_t groups = (a.tokens + TOKENS - 1) / TOKENS;
  // A thread for each of a token's pieces; where tokens are few, workgroups of 128 threads for them (in place of up to
  // 1024: 4 tokens of 256 bf16 heads of 128 2.7 us for 3.6, 8 of 192 to an e4m3 cache 3.3 for 4.6, 200 of 40 the same).
  const int most = groups < 256 ? kFewThreads : kMaxThreads;
  const int threads = (of_token + 63) / 64 * 64 < most ? (of_token + 63) / 64 * 64 : most;
  const int slices = groups < 256 ? (of_token + threads - 1) / threads : 1;
  const dim3 grid((unsigned)(groups < kMaxGroups ? groups : kMaxGroups), (unsigned)slices);
  rope_at<C, KC, INTERLEAVED, CACHE, WHOLE, NT, TOKENS>
      <<<grid, threads, (size_t)TOKENS * a.half * sizeof(f32x2), st>>>(a, copy_q ? 1 : 0);
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
  if (of_token > (int64_t(1) << 21)) return (int32_t)hipErrorInvalidValue;  // a token's pieces are counted in 32 bits
  if (of_token == 0) return (int32_t)hipSuccess;
  if (!whole) return run<C, KC, INTERLEAVED, CACHE, false, false, 1>(a, copy_q, (int)of_token, st);
  const int64_t bytes = a.tokens * (a.q.heads + a.k.heads) * a.dim * C::kBytes;
  // 32-bit offsets in a token, of tensors that go past the caches (bf16, 40 heads of 128, us, so and not: 4096 tokens,
  // 42 MB, 16.9 and 15.2; 8192 29.4 and 29.4; 16384 54.3 and 59.8; 32768 105 and 114). With a cache two tokens a
  // workgroup (8192 tokens 40.9, one 43.2), without one (32768 tokens 105, two 109).
  const auto reach = [&](const Heads& h) {
    return h.to_head >= 0 && (h.heads * h.to_head + a.dim) * C::kBytes <= INT32_MAX;
  };
  if (bytes >= (int64_t(1) << 26) && reach(a.q) && reach(a.k)) {
    return run<C, KC, INTERLEAVED, CACHE, true, true, CACHE ? 2 : 1>(a, copy_q, (int)of_token, st);
  }
  return run<C, KC, INTERLEAVED, CACHE, true, false, 1>(a, copy_q, (int)of_token, st);
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
    return interleaved ? by_shape<C, Plain<C>, true, false>(a, copy, st)
                       : by_shape<C, Plain<C>, false, false>(a, copy, st);
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
    return run_to(Plain<C>{});
  });
}

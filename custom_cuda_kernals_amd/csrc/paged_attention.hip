// Attention of one new token a sequence over a paged key-value cache.
//
//   s_j = scale q . k_j     p_j = exp(s_j) / sum exp(s_j)     out = sum p_j v_j
//
// over the positions j of a sequence that its page table has a page for; lse = log sum
// exp(s_j). One pass with a running maximum and sum, in float32. The G query heads of one
// key-value head are the columns of the matrix instructions, so their keys and values
// are read once:
//
//   S^T [16 positions][G] = K Q^T       keys as they lie in memory
//   O^T [16 elements][G] += V^T P^T     values turned over in LDS
//
// A lane's four scores of a tile are of its own column and of the positions its operand of
// the second product wants (the order of the contracted positions is free), so P goes from
// one product to the other inside the lane. 16-bit P is split in two parts, high and low:
// rounded once, it would add an error as large as that of the output's own rounding.
//
// Bound by HBM: reading keys and values once. A sequence is cut into as many parts as fill
// the card; a workgroup takes a part of one key-value head, its four waves every fourth
// step of it, each on its own until the sums of the waves meet in LDS. The parts' sums
// meet in a second launch.
#include "tile_product.hpp"

namespace cck {
namespace {

constexpr int kWaves = 4, kHeads = 16;  // of a workgroup: waves, and query heads at most
constexpr int kMinPart = 128;           // positions of a part, at least: a step of each wave
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// Sums are scaled to a new maximum only where it is this much (a power of two) above the
// one that they have.
constexpr float kSlack = 8.0f;

struct AttentionArgs {
  const char *q, *keys, *values;
  const int64_t *table, *lengths;
  char* out;
  float *lse, *partial;  // partial: [sequence][key-value head][part][G][dim], then [..][G][2]
  int64_t q_token, q_head, pages;
  int sequences, heads, kv_heads, dim, page, table_width, window, parts, head_tiles;
  uint32_t page_magic;
  int page_shift;
  float score_scale, value_scale;  // score_scale: with log2(e)
};

// What the elements of a head's row are computed in. A chunk is what a lane loads of a
// row: 16 bytes.
struct Bf16 {
  using Codec = CodecBF16;
  static constexpr int kBytes = 2;
  __device__ static f32x4 mma(const u32x4& a, const u32x4& b, const f32x4& c) { return ElemBF16::mma(a, b, c, 0, 0); }
  __device__ static uint32_t pack(float lo, float hi) { return pack2_bf16(lo, hi); }
  __device__ static float low(uint32_t w) { return bf16_lo(w); }
  __device__ static float high(uint32_t w) { return bf16_hi(w); }
};
struct F16 {
  using Codec = CodecF16;
  static constexpr int kBytes = 2;
  __device__ static f32x4 mma(const u32x4& a, const u32x4& b, const f32x4& c) { return ElemF16::mma(a, b, c, 0, 0); }
  __device__ static uint32_t pack(float lo, float hi) { return pack2_f16(lo, hi); }
  __device__ static float low(uint32_t w) { return f16_lo(w); }
  __device__ static float high(uint32_t w) { return f16_hi(w); }
};
struct F32 {
  using Codec = CodecF32;
  static constexpr int kBytes = 4;
  __device__ static f32x4 mma(const u32x4& a, const u32x4& b, const f32x4& c) { return ElemF32::mma(a, b, c, 0, 0); }
};

// How a chunk in memory becomes fragments of T: kFragments of 16 bytes.
template <class T>
struct AsIs {
  static constexpr int kFragments = 1, kBytes = T::kBytes;
  __device__ static void fragments(const u32x4& w, u32x4 (&f)[1]) { f[0] = w; }
};
// FP8 codes are exact in 16 bits: their scale is applied to the sums.
template <class T, int FMT>
struct FromCodes {
  static constexpr int kFragments = T::kBytes, kBytes = 1;
  __device__ static f32x2 two(uint32_t w, bool high) {
    if constexpr (FMT == kF8E4M3) {
      return high ? __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true) : __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
    } else {
      return high ? __builtin_amdgcn_cvt_pk_f32_bf8((int)w, true) : __builtin_amdgcn_cvt_pk_f32_bf8((int)w, false);
    }
  }
  __device__ static void fragments(const u32x4& w, u32x4 (&f)[kFragments]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x2 a = two(w[i], false), b = two(w[i], true);
      if constexpr (T::kBytes == 2) {
        f[i / 2][i % 2 * 2] = T::pack(a[0], a[1]);
        f[i / 2][i % 2 * 2 + 1] = T::pack(b[0], b[1]);
      } else {
        f[i] = (u32x4){f32_bits(a[0]), f32_bits(a[1]), f32_bits(b[0]), f32_bits(b[1])};
      }
    }
  }
};

// Positions [lo, hi) of a sequence that are seen, and of one of its parts; count: its parts.
struct Span {
  int lo, hi, begin, end, count;
  __device__ Span(const AttentionArgs& a, int sequence, int part) {
    const int64_t most = (int64_t)a.table_width * a.page;
    int64_t n = a.lengths[sequence];
    n = n < 0 ? 0 : n > most ? most : n;
    hi = __builtin_amdgcn_readfirstlane((int)n);
    lo = a.window > 0 && hi > a.window ? hi - a.window : 0;
    const int seen = hi - lo;
    int each = (seen + a.parts - 1) / a.parts;
    each = (each + kMinPart - 1) / kMinPart * kMinPart;
    each = each < kMinPart ? kMinPart : each;
    count = (seen + each - 1) / each;
    begin = lo + part * each;
    end = begin + each < hi ? begin + each : hi;
  }
};

// LDS bytes of a row of values: an odd multiple of 32, so that eight rows begin in
// different banks.
constexpr __host__ __device__ int row_bytes(int elements, int bytes) { return ((elements * bytes + 31) / 32 | 1) * 32; }

// DIM: the head's elements, padded. A step: kStep positions of a wave.
template <class T, class S, int DIM>
struct Shape {
  static constexpr int kTiles = T::kBytes == 4 ? 1 : 2, kStep = 16 * kTiles;
  static constexpr int kElements = 16 / S::kBytes;             // of a chunk
  static constexpr int kChunks = (DIM + 4 * kElements - 1) / (4 * kElements);  // of a lane and row
  static constexpr int kRow = row_bytes(DIM, T::kBytes);
  static constexpr int kWaveLds = kStep * kRow;
  static constexpr int kSumsLds = kHeads * DIM * 4;
  static constexpr int kLds = kWaves * (kWaveLds > kSumsLds ? kWaveLds : kSumsLds);
};

template <class T, class S, int DIM>
__global__ __launch_bounds__(kWaves * 64, T::kBytes == 2 && DIM <= 128 ? 2 : 1) void paged_attention(AttentionArgs a) {
  using Sh = Shape<T, S, DIM>;
  constexpr int kTiles = Sh::kTiles, kStep = Sh::kStep, kChunks = Sh::kChunks, kFrags = S::kFragments, kRow = Sh::kRow;
  __shared__ __attribute__((aligned(64))) char lds[Sh::kLds];
  __shared__ float stats[kWaves][kHeads][2];

  const int units = a.kv_heads * a.head_tiles;
  int id = blockIdx.x;
  const int unit = id % units;
  id /= units;
  const int sequence = id % a.sequences, part = id / a.sequences;
  const int kv = unit / a.head_tiles, group = a.heads / a.kv_heads;
  const int head0 = unit % a.head_tiles * kHeads, heads = group - head0 < kHeads ? group - head0 : kHeads;
  const Span span(a, sequence, part);
  if (part >= span.count && part > 0) return;

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int col = lane & 15, g = lane >> 4;
  const LdsPtr mine = (LdsPtr)lds + wave * Sh::kWaveLds;

  // The columns' queries: of each chunk of a row the elements that this lane has.
  u32x4 q[kChunks][kFrags];
  {
    const int h = kv * group + head0 + (col < heads ? col : 0);
    const char* from = a.q + ((int64_t)sequence * a.q_token + (int64_t)h * a.q_head) * T::kBytes;
#pragma unroll
    for (int s = 0; s < kChunks; ++s) {
#pragma unroll
      for (int f = 0; f < kFrags; ++f) {
        const int e = (4 * s + g) * Sh::kElements + f * (16 / T::kBytes);
        q[s][f] = (u32x4){0u, 0u, 0u, 0u};
        if (e < a.dim) q[s][f] = *reinterpret_cast<const u32x4_any*>(from + e * T::kBytes);
      }
    }
  }

  const int64_t* table = a.table + (int64_t)sequence * a.table_width;
  const int64_t slot_bytes = (int64_t)a.kv_heads * a.dim * S::kBytes;
  const int64_t head_bytes = (int64_t)kv * a.dim * S::kBytes;
  // Where the lane's positions of a step lie: slots, or -1 for none.
  auto find = [&](int first, int64_t (&slot)[kTiles]) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < kTiles; ++j) {
      const int t = first + 16 * j + col;
      slot[j] = -1;
      if (t < span.end) {
        const uint32_t at = (uint32_t)(((uint64_t)(uint32_t)t * a.page_magic) >> a.page_shift);
        const int64_t page = table[at];
        if (page >= 0 && page < a.pages) slot[j] = page * a.page + (t - (int)at * a.page);
      }
    }
  };
  const int row = a.dim * S::kBytes;
  u32x4 k[kTiles][kChunks], v[kTiles][kChunks];
  auto load = [&](const int64_t (&slot)[kTiles]) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < kTiles; ++j) {
      const int64_t at = (slot[j] < 0 ? 0 : slot[j]) * slot_bytes + head_bytes;
#pragma unroll
      for (int s = 0; s < kChunks; ++s) {
        const int byte = (4 * s + g) * 16, last = row - 16;  // past the row its last chunk will do
        k[j][s] = *reinterpret_cast<const u32x4_any*>(a.keys + at + (byte < last ? byte : last));
        v[j][s] = *reinterpret_cast<const u32x4_any*>(a.values + at + (byte < last ? byte : last));
      }
    }
  };

  constexpr int kOut = DIM / 16;
  f32x4 out[kOut] = {};
  float top = -__builtin_inff(), base = 0.0f, sum = 0.0f;  // base: top, or 0 while there is none
  int64_t slot[kTiles], next_slot[kTiles];
  int first = span.begin + wave * kStep;
  find(first, slot);
  if (first < span.end) load(slot);
  find(first + kWaves * kStep, next_slot);
  for (; first < span.end; first += kWaves * kStep) {
    // Values to LDS, those of positions that are not seen as zeros.
    uint64_t seen[kTiles];
    bool all = true;
#pragma unroll
    for (int j = 0; j < kTiles; ++j) {
      seen[j] = __ballot(slot[j] >= 0);
      all = all && seen[j] == ~0ull;
    }
#pragma unroll
    for (int j = 0; j < kTiles; ++j) {
#pragma unroll
      for (int s = 0; s < kChunks; ++s) {
        u32x4 w = v[j][s];
        if (!all && slot[j] < 0) w = (u32x4){0u, 0u, 0u, 0u};
        u32x4 f[kFrags];
        S::fragments(w, f);
        const int e = (4 * s + g) * Sh::kElements;
        if (DIM % (4 * Sh::kElements) == 0 || e < DIM) {
#pragma unroll
          for (int i = 0; i < kFrags; ++i) lds_store(f[i], mine + (16 * j + col) * kRow + e * T::kBytes + i * 16);
        }
      }
    }
    f32x4 score[kTiles] = {};
#pragma unroll
    for (int j = 0; j < kTiles; ++j) {
#pragma unroll
      for (int s = 0; s < kChunks; ++s) {
        u32x4 w = k[j][s], f[kFrags];
        if ((4 * s + 4) * 16 > row && (4 * s + g) * 16 >= row) w = (u32x4){0u, 0u, 0u, 0u};
        S::fragments(w, f);
#pragma unroll
        for (int i = 0; i < kFrags; ++i) score[j] = T::mma(f[i], q[s][i], score[j]);
      }
    }
    // The next step's.
#pragma unroll
    for (int j = 0; j < kTiles; ++j) slot[j] = next_slot[j];
    if (first + kWaves * kStep < span.end) load(slot);
    find(first + 2 * kWaves * kStep, next_slot);

    float most = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < kTiles; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x = score[j][i] * a.score_scale;
        if (!all && !(seen[j] >> (4 * g + i) & 1)) x = -__builtin_inff();
        score[j][i] = x;
        most = __builtin_fmaxf(most, x);
      }
    }
    if (__any(most > top + kSlack)) {
      most = __builtin_fmaxf(most, __shfl_xor(most, 16));
      most = __builtin_fmaxf(most, __shfl_xor(most, 32));
      const float now = __builtin_fmaxf(top, most);
      base = now == -__builtin_inff() ? 0.0f : now;
      const float keep = __builtin_amdgcn_exp2f(top - base);
      top = now;
      sum *= keep;
#pragma unroll
      for (int f = 0; f < kOut; ++f) out[f] *= keep;
    }
#pragma unroll
    for (int j = 0; j < kTiles; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        score[j][i] = __builtin_amdgcn_exp2f(score[j][i] - base);
        sum += score[j][i];
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if constexpr (T::kBytes == 2) {
      u32x4 high, low;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float x = score[j][2 * i], y = score[j][2 * i + 1];
          const uint32_t h = T::pack(x, y);
          high[2 * j + i] = h;
          low[2 * j + i] = T::pack(x - T::low(h), y - T::high(h));
        }
      }
      // Four rows of 16 elements, turned over: row 4 g + lane / 4 % 4 of a tile.
      using Lds4 = __attribute__((address_space(3))) s16x4*;
      const LdsPtr from = mine + (4 * g + (col >> 2)) * kRow + (col & 3) * 8;
#pragma unroll
      for (int f = 0; f < kOut; ++f) {
        if (16 * f < a.dim) {
          const u32x2 x = __builtin_bit_cast(
              u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<Lds4>(from + f * 32)));
          const u32x2 y = __builtin_bit_cast(
              u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<Lds4>(from + f * 32 + 16 * kRow)));
          const u32x4 w = {x[0], x[1], y[0], y[1]};
          out[f] = T::mma(w, high, out[f]);
          out[f] = T::mma(w, low, out[f]);
        }
      }
    } else {
      const u32x4 p = __builtin_bit_cast(u32x4, score[0]);
#pragma unroll
      for (int f = 0; f < kOut; ++f) {
        if (16 * f < a.dim) {
          u32x4 w;
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = lds_load<uint32_t>(mine + (4 * g + i) * kRow + (16 * f + col) * 4);
          out[f] = T::mma(w, p, out[f]);
        }
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
  sum += __shfl_xor(sum, 16);
  sum += __shfl_xor(sum, 32);

  // The waves' sums meet: [wave][head][dim] in LDS.
  __syncthreads();
  float* const sums = reinterpret_cast<float*>(lds);
  if (g == 0) {
    stats[wave][col][0] = top;
    stats[wave][col][1] = sum;
  }
#pragma unroll
  for (int f = 0; f < kOut; ++f) {
    *reinterpret_cast<f32x4*>(sums + (wave * kHeads + col) * DIM + 16 * f + 4 * g) = out[f];
  }
  __syncthreads();
  const int quads = a.dim / 4;
  for (int i = threadIdx.x; i < heads * quads; i += kWaves * 64) {
    const int h = i / quads, d = (i - h * quads) * 4;
    float all_top = stats[0][h][0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) all_top = __builtin_fmaxf(all_top, stats[w][h][0]);
    const float all_base = all_top == -__builtin_inff() ? 0.0f : all_top;
    float total = 0.0f;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float weight = __builtin_amdgcn_exp2f(stats[w][h][0] - all_base);
      total += weight * stats[w][h][1];
      o += weight * *reinterpret_cast<const f32x4*>(sums + (w * kHeads + h) * DIM + d);
    }
    const int64_t head = (int64_t)sequence * a.heads + kv * group + head0 + h;
    if (a.parts > 1) {
      const int64_t row = head * a.parts + part;
      *reinterpret_cast<f32x4*>(a.partial + row * a.dim + d) = o;
      if (d == 0) {
        float* const at = a.partial + (int64_t)a.sequences * a.heads * a.parts * a.dim + row * 2;
        at[0] = all_top;
        at[1] = total;
      }
    } else {
      const float inverse = total == 0.0f ? 0.0f : a.value_scale / total;
#pragma unroll
      for (int j = 0; j < 4; ++j) T::Codec::store1(a.out, head * a.dim + d + j, total == 0.0f ? 0.0f : o[j] * inverse);
      if (d == 0 && a.lse != nullptr) {
        a.lse[head] = total == 0.0f ? -__builtin_inff() : (all_top + __builtin_log2f(total)) * kLn2;
      }
    }
  }
}

// The parts' sums, a head a workgroup.
template <class C>
__global__ __launch_bounds__(256) void join_parts(AttentionArgs a) {
  __shared__ float weights[256];
  __shared__ f32x4 sums[256];
  const int64_t head = blockIdx.x;
  const Span span(a, (int)(head / a.heads), 0);
  const int count = span.count, tid = threadIdx.x;
  const float* const stats = a.partial + (int64_t)a.sequences * a.heads * a.parts * a.dim + head * a.parts * 2;
  float top = -__builtin_inff();
  for (int i = tid & 63; i < count; i += 64) top = __builtin_fmaxf(top, stats[2 * i]);
#pragma unroll
  for (int d = 1; d < 64; d *= 2) top = __builtin_fmaxf(top, __shfl_xor(top, d));
  const float base = top == -__builtin_inff() ? 0.0f : top;
  float total = 0.0f;
  for (int i = tid & 63; i < count; i += 64) {
    const float w = __builtin_amdgcn_exp2f(stats[2 * i] - base);
    total += w * stats[2 * i + 1];
    if (tid < 64 && i < 256) weights[i] = w;
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) total += __shfl_xor(total, d);
  __syncthreads();
  // Threads of one quad of elements take every `lanes`-th part.
  const int quads = a.dim / 4, lanes = 256 / quads, quad = tid % quads, of = tid / quads;
  f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  if (of < lanes) {
    const float* from = a.partial + head * a.parts * a.dim + quad * 4;
    for (int i = of; i < count; i += lanes) o += weights[i] * *reinterpret_cast<const f32x4*>(from + (int64_t)i * a.dim);
  }
  sums[tid] = o;
  __syncthreads();
  if (tid < quads) {
    for (int i = 1; i < lanes; ++i) o += sums[i * quads + tid];
    const float inverse = total == 0.0f ? 0.0f : a.value_scale / total;
#pragma unroll
    for (int j = 0; j < 4; ++j) C::store1(a.out, head * a.dim + tid * 4 + j, total == 0.0f ? 0.0f : o[j] * inverse);
    if (tid == 0 && a.lse != nullptr) {
      a.lse[head] = total == 0.0f ? -__builtin_inff() : (top + __builtin_log2f(total)) * kLn2;
    }
  }
}

constexpr int kMaxParts = 256;  // join_parts holds a weight for each
constexpr int64_t kMaxPositions = int64_t(1) << 30;  // of a sequence: a step past the last is still an int

int head_tiles_of(int64_t heads, int64_t kv_heads) { return (int)((heads / kv_heads + kHeads - 1) / kHeads); }

// Parts of a sequence: as many as make 2048 workgroups, of kMinPart positions at least.
int parts_of(int64_t sequences, int64_t units, int64_t positions) {
  const int64_t groups = sequences * units, wanted = (2048 + groups - 1) / groups;
  const int64_t most = (positions + kMinPart - 1) / kMinPart;
  int64_t parts = wanted < most ? wanted : most;
  parts = parts < kMaxParts ? parts : kMaxParts;
  return (int)(parts < 1 ? 1 : parts);
}

template <class T, class S>
int32_t run_dim(const AttentionArgs& a, int64_t blocks, hipStream_t st) {
  if (a.dim <= 64) {
    paged_attention<T, S, 64><<<(unsigned)blocks, kWaves * 64, 0, st>>>(a);
  } else if (a.dim <= 128) {
    paged_attention<T, S, 128><<<(unsigned)blocks, kWaves * 64, 0, st>>>(a);
  } else {
    paged_attention<T, S, 256><<<(unsigned)blocks, kWaves * 64, 0, st>>>(a);
  }
  int32_t status = launch_status();
  if (status == 0 && a.parts > 1) {
    join_parts<typename T::Codec><<<(unsigned)(a.sequences * a.heads), 256, 0, st>>>(a);
    status = launch_status();
  }
  return status;
}

template <class T>
int32_t run_cache(const AttentionArgs& a, int64_t blocks, int32_t cache_dtype, hipStream_t st) {
  if (cache_dtype == kF8E4M3) return run_dim<T, FromCodes<T, kF8E4M3>>(a, blocks, st);
  if (cache_dtype == kF8E5M2) return run_dim<T, FromCodes<T, kF8E5M2>>(a, blocks, st);
  return run_dim<T, AsIs<T>>(a, blocks, st);
}

bool attention_sizes_ok(int64_t sequences, int64_t heads, int64_t kv_heads, int64_t dim, int64_t page,
                        int64_t table_width) {
  return kv_heads >= 1 && heads >= kv_heads && heads % kv_heads == 0 && heads <= 65536 && dim >= 16 && dim <= 256 &&
         dim % 16 == 0 && page >= 1 && table_width >= 0 && table_width <= kMaxPositions / page &&
         sequences <= (int64_t(1) << 23) / heads;
}

}  // namespace
}  // namespace cck

using namespace cck;

extern "C" int64_t cck_paged_attention_workspace(int64_t sequences, int64_t n_q_heads, int64_t n_kv_heads,
                                                 int64_t head_dim, int64_t page_size, int64_t table_width) {
  if (sequences <= 0 || !attention_sizes_ok(sequences, n_q_heads, n_kv_heads, head_dim, page_size, table_width)) return 0;
  const int parts = parts_of(sequences, n_kv_heads * head_tiles_of(n_q_heads, n_kv_heads), page_size * table_width);
  return parts == 1 ? 0 : sequences * n_q_heads * parts * (head_dim + 2) * 4;
}

extern "C" int32_t launch_paged_attention_fwd(const void* q, const void* key_cache, const void* value_cache,
                                              const int64_t* page_table, const int64_t* lengths, void* out, float* lse,
                                              void* workspace, int64_t q_token_stride, int64_t q_head_stride,
                                              int64_t sequences, int64_t n_q_heads, int64_t n_kv_heads,
                                              int64_t head_dim, int64_t pages, int64_t page_size, int64_t table_width,
                                              int64_t window, float scale, float key_scale, float value_scale,
                                              int32_t dtype, int32_t cache_dtype, void* stream) {
  if (dtype != kF32 && dtype != kF16 && dtype != kBF16) return (int32_t)hipErrorInvalidValue;
  if (cache_dtype != dtype && cache_dtype != kF8E4M3 && cache_dtype != kF8E5M2) return (int32_t)hipErrorInvalidValue;
  if (sequences <= 0 || n_q_heads <= 0) return (int32_t)hipSuccess;
  if (!attention_sizes_ok(sequences, n_q_heads, n_kv_heads, head_dim, page_size, table_width) || pages < 0 ||
      pages > INT64_MAX / page_size / n_kv_heads / head_dim / 4) {
    return (int32_t)hipErrorInvalidValue;
  }
  AttentionArgs a = {};
  a.q = static_cast<const char*>(q);
  a.keys = static_cast<const char*>(key_cache);
  a.values = static_cast<const char*>(value_cache);
  a.table = page_table;
  a.lengths = lengths;
  a.out = static_cast<char*>(out);
  a.lse = lse;
  a.partial = static_cast<float*>(workspace);
  a.q_token = q_token_stride;
  a.q_head = q_head_stride;
  a.pages = pages;
  a.sequences = (int)sequences;
  a.heads = (int)n_q_heads;
  a.kv_heads = (int)n_kv_heads;
  a.dim = (int)head_dim;
  a.page = (int)page_size;
  a.table_width = pages > 0 ? (int)table_width : 0;  // no page: no position
  a.window = window > 0 && window < INT32_MAX ? (int)window : 0;
  a.head_tiles = head_tiles_of(n_q_heads, n_kv_heads);
  a.parts = parts_of(sequences, n_kv_heads * a.head_tiles, page_size * table_width);
  if (a.parts > 1 && (workspace == nullptr || !host_aligned(workspace, 16))) return (int32_t)hipErrorInvalidValue;
  // t / page for t < 2^31: t * magic >> shift, magic = floor(2^(31 + bits) / page) + 1 with
  // 2^bits >= page. What magic is too large by, at most 1, adds less than 2^-bits <= 1 / page.
  int bits = 0;
  while ((int64_t(1) << bits) < page_size) ++bits;
  a.page_shift = 31 + bits;
  a.page_magic = (uint32_t)(((unsigned __int128)1 << (31 + bits)) / (uint64_t)page_size + 1);
  a.score_scale = scale * key_scale * kLog2e;
  a.value_scale = value_scale;
  const int64_t blocks = sequences * n_kv_heads * a.head_tiles * a.parts;
  if (blocks > (int64_t(1) << 24) - 1) return (int32_t)hipErrorInvalidValue;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case kF32: return run_cache<F32>(a, blocks, cache_dtype, st);
    case kF16: return run_cache<F16>(a, blocks, cache_dtype, st);
    default: return run_cache<Bf16>(a, blocks, cache_dtype, st);
  }
}

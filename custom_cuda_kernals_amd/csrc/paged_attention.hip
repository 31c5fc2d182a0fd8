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
// Bound by HBM: reading keys and values once. A wave works alone, on positions of one
// sequence and one key-value head. Short contexts have a wave or a workgroup's few waves
// for each; long ones are cut into parts of one length, as many as fill the card, whose
// sums meet in a second launch. The lengths are on the GPU, so each workgroup finds its
// part itself, from the sum of all lengths. Keys and values go straight from memory to
// LDS, whole rows at a time, into a ring of two steps or more: steps are on their way
// while one is worked on, without registers or other waves to wait for.
//
// 8 key-value heads of 128: 64 sequences of up to 8192 positions, bf16, 1.08 GB, 192 us,
// 5.6 TB/s (a copy of 1 GiB reaches 5.2, one of 320 MiB 6.7); two of 131072, e4m3, 0.54 GB,
// 111 us, 4.8 TB/s; 1024 of up to 512 181 us, 5.9 TB/s; one of 700 10.3 us, where steps are
// waited for. Worst: many short sequences in wide tables, as all parts read all lengths
// (2048 of up to 100 positions 539 us in tables for 8192, 108 in tables for 112).
#include "tile_product.hpp"

namespace cck {
namespace {

constexpr int kHeads = 16;    // query heads of a workgroup, at most
constexpr int kMinPart = 32;  // positions of a part, at least: a step
constexpr int kFound = 512;   // positions whose slots are looked up at a time
constexpr int kRing = 32768;  // bytes of LDS for the steps of a wave: more only if two steps need it
constexpr int kMaxCut = 2048;  // sequences: beyond it each is one part, so that nobody reads so many lengths
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// Sums are scaled to a new maximum only where it is this much (a power of two) above the
// one that they have.
constexpr float kSlack = 8.0f;
// The power of two of P where sums passed float32's range: 2^30 values below 2^128 stay below 2^126.
constexpr int kDown = -40;

struct AttentionArgs {
  const char *q, *keys, *values;
  const int64_t *table, *lengths;
  char* out;
  // partial: [parts][heads][dim], then [parts][heads][2], the maximum and the sum, and then of each sequence
  // its first part and how many it has.
  float *lse, *partial;
  int64_t q_token, q_head, pages;
  int sequences, heads, kv_heads, dim, page, table_width, window, head_tiles;
  int parts;  // of all sequences together, at most; 0: each sequence is one
  uint32_t page_magic;
  int page_shift;
  float score_scale, value_scale;  // score_scale: with log2(e)
  float part_cost;                 // kPartCost for each of the places, or 0: see parts_of
};

using i32x2 = int __attribute__((ext_vector_type(2)));

// What the elements of a head's row are computed in. A chunk is what a lane loads of a
// row: 16 bytes.
struct Bf16 {
  using Codec = CodecBF16;
  static constexpr int kBytes = 2, kLift = 0, kLiftAgain = kDown;
  static constexpr uint32_t kInfinity = 0x7f80u;
  __device__ static f32x4 mma(const u32x4& a, const u32x4& b, const f32x4& c) { return ElemBF16::mma(a, b, c, 0, 0); }
  __device__ static uint32_t pack(float lo, float hi) { return pack2_bf16(lo, hi); }
  __device__ static float low(uint32_t w) { return bf16_lo(w); }
  __device__ static float high(uint32_t w) { return bf16_hi(w); }
};
struct F16 {
  using Codec = CodecF16;
  // P times 2^7: with kSlack 2^15 at most, and what a long tail of small ones has keeps its bits down to 2^-31.
  static constexpr int kBytes = 2, kLift = 7, kLiftAgain = 7;
  static constexpr uint32_t kInfinity = 0x7c00u;
  __device__ static f32x4 mma(const u32x4& a, const u32x4& b, const f32x4& c) { return ElemF16::mma(a, b, c, 0, 0); }
  __device__ static uint32_t pack(float lo, float hi) { return pack2_f16(lo, hi); }
  __device__ static float low(uint32_t w) { return f16_lo(w); }
  __device__ static float high(uint32_t w) { return f16_hi(w); }
};
struct F32 {
  using Codec = CodecF32;
  static constexpr int kBytes = 4, kLift = 0, kLiftAgain = kDown;
  static constexpr uint32_t kInfinity = 0x7f800000u;
  __device__ static f32x4 mma(const u32x4& a, const u32x4& b, const f32x4& c) { return ElemF32::mma(a, b, c, 0, 0); }
};

// The infinite elements and those that are no numbers, zeros for the others.
template <class T>
__device__ inline u32x4 not_finite(u32x4 w) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (T::kBytes == 4) {
      w[i] = (w[i] & T::kInfinity) == T::kInfinity ? w[i] : 0u;
    } else {
      const uint32_t low = (w[i] & T::kInfinity) == T::kInfinity ? w[i] & 0xffffu : 0u;
      const uint32_t high = (w[i] >> 16 & T::kInfinity) == T::kInfinity ? w[i] & 0xffff0000u : 0u;
      w[i] = low | high;
    }
  }
  return w;
}
// Whether all are: 0 x is NaN if x is not. One comparison in the end, where one each took 0.3 us.
template <int N>
__device__ inline bool finite(const f32x4 (&v)[N]) {
  f32x4 zero = v[0] * 0.0f;
#pragma unroll
  for (int f = 1; f < N; ++f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) zero[i] = __builtin_fmaf(v[f][i], 0.0f, zero[i]);
  }
  return (zero[0] + zero[1]) + (zero[2] + zero[3]) == 0.0f;
}
__device__ inline bool finite(const f32x4& v) {
  const f32x4 one[1] = {v};
  return finite(one);
}

// A part's sums to those of all, by 2^kDown: where the sums of parts pass float32's range.
__device__ inline void add_down(f32x4& o, float& total, const f32x4& part, const f32x2& stat, float base) {
  const float p = __builtin_amdgcn_exp2f(stat[0] - base), down = __builtin_ldexpf(p, kDown);
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] += (__builtin_fabsf(part[i]) < __builtin_inff() ? down : p) * part[i];
  total += down * stat[1];
}

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
  // Four codes to four elements, of 16 or 32 bits.
  __device__ static void four(uint32_t w, uint32_t (&e)[T::kBytes]) {
    if constexpr (T::kBytes == 4) {
      const f32x2 a = FMT == kF8E4M3 ? __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false) : __builtin_amdgcn_cvt_pk_f32_bf8((int)w, false);
      const f32x2 b = FMT == kF8E4M3 ? __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true) : __builtin_amdgcn_cvt_pk_f32_bf8((int)w, true);
      e[0] = f32_bits(a[0]), e[1] = f32_bits(a[1]), e[2] = f32_bits(b[0]), e[3] = f32_bits(b[1]);
    } else if constexpr (std::is_same_v<T, Bf16>) {
      e[0] = __builtin_bit_cast(uint32_t, FMT == kF8E4M3 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false)
                                                         : __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w, 1.0f, false));
      e[1] = __builtin_bit_cast(uint32_t, FMT == kF8E4M3 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true)
                                                         : __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w, 1.0f, true));
    } else {
      e[0] = __builtin_bit_cast(uint32_t, FMT == kF8E4M3 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false)
                                                         : __builtin_amdgcn_cvt_scalef32_pk_f16_bf8(w, 1.0f, false));
      e[1] = __builtin_bit_cast(uint32_t, FMT == kF8E4M3 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true)
                                                         : __builtin_amdgcn_cvt_scalef32_pk_f16_bf8(w, 1.0f, true));
    }
  }
  __device__ static void fragments(const u32x4& w, u32x4 (&f)[kFragments]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t e[T::kBytes];
      four(w[i], e);
#pragma unroll
      for (int j = 0; j < T::kBytes; ++j) f[(i * T::kBytes + j) / 4][(i * T::kBytes + j) % 4] = e[j];
    }
  }
};

// The positions of a sequence that are seen: [lo, lo + seen).
struct Seen {
  int lo = 0, seen = 0;
  __device__ Seen() = default;
  // Of n positions.
  __device__ Seen(const AttentionArgs& a, int n) {
    lo = a.window > 0 && n > a.window ? n - a.window : 0;
    seen = n - lo;
  }
  __device__ static int in_table(const AttentionArgs& a, int64_t n) {
    const int64_t most = (int64_t)a.table_width * a.page;
    return (int)(n < 0 ? 0 : n > most ? most : n);
  }
  __device__ static Seen of(const AttentionArgs& a, int sequence) {
    return Seen(a, in_table(a, a.lengths[sequence]));
  }
};

__device__ inline float* stats_of(const AttentionArgs& a) { return a.partial + (int64_t)a.parts * a.heads * a.dim; }
__device__ inline int* notes_of(const AttentionArgs& a) {
  return reinterpret_cast<int*>(stats_of(a) + (int64_t)a.parts * a.heads * 2);
}

// How the sequences are cut: into parts of `each` positions, numbered through all of them.
// A lane has a run of sequences, and knows how many parts come before them. Every lane of
// the wave calls. The lengths of runs of more than one wait in `room`, in LDS.
struct Cut {
  int each, run, mine, before, all;  // sequences of a run; parts of the lane's, before them, and of all
  Seen only;                         // of a lane's one sequence
  const int* lengths;
  __device__ Cut(const AttentionArgs& a, int* room) : run((a.sequences + 63) / 64), lengths(room) {
    const int first = (int)(threadIdx.x & 63) * run;
    double total = 0.0;  // exact: below 2^41
    if (run == 1) {
      if (first < a.sequences) only = Seen::of(a, first);
      total = (double)only.seen;
    } else {
      constexpr int kAtOnce = 8;
      for (int i = (int)(threadIdx.x & 63); i < a.sequences; i += 64 * kAtOnce) {
        int64_t n[kAtOnce];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) n[u] = a.lengths[i + 64 * u < a.sequences ? i + 64 * u : i];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
          if (i + 64 * u < a.sequences) room[i + 64 * u] = Seen::in_table(a, n[u]);
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      for (int i = 0; i < run; ++i) {
        if (first + i < a.sequences) total += (double)Seen(a, lengths[first + i]).seen;
      }
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) total += __shfl_xor(total, d);
    // Each sequence has a last part that may be short, so that there are no more than a.parts in all.
    // The host has allowed for as many as the table has room for; what the lengths call for may be fewer.
    const double even = total / (double)(a.parts - a.sequences), worth = __builtin_sqrt(total * a.part_cost);
    const int wanted = (int)__builtin_ceil(even > worth ? even : worth);
    each = __builtin_amdgcn_readfirstlane((wanted + kMinPart - 1) / kMinPart * kMinPart);
    each = each < kMinPart ? kMinPart : each;
    mine = 0;
    for (int i = 0; i < run; ++i) mine += parts_of(a, first + i);
    int sum = mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int v = __shfl_up(sum, d);
      if ((int)(threadIdx.x & 63) >= d) sum += v;
    }
    before = sum - mine;
    all = __builtin_amdgcn_readlane(sum, 63);
  }
  // Of one of the lane's sequences.
  __device__ int parts_of(const AttentionArgs& a, int sequence) const {
    if (run == 1) return (only.seen + each - 1) / each;  // the lane's; 0 behind the last sequence
    return sequence < a.sequences ? (Seen(a, lengths[sequence]).seen + each - 1) / each : 0;
  }
  // First part and number of parts of each sequence, for the launch that joins them.
  __device__ void note(const AttentionArgs& a) const {
    int* const notes = notes_of(a);
    int at = before;
    for (int i = 0; i < run; ++i) {
      const int s = (int)(threadIdx.x & 63) * run + i, n = parts_of(a, s);
      if (s < a.sequences) {
        notes[2 * s] = at;
        notes[2 * s + 1] = n;
      }
      at += n;
    }
  }
};

// A workgroup's work: positions [begin, end) of a sequence that has `count` parts, and which
// heads. All heads of a part go to one XCD, one after another. In turn they would go to the
// XCDs in turn too, and an XCD then read the same few hundred bytes of each row of heads,
// which are the same few channels of its L2.
struct Part {
  int index = 0, unit = 0, sequence = 0, begin = 0, end = 0, count = 1;
  bool none = false;
  __device__ Part(const AttentionArgs& a, int id, int* room) {
    const int units = a.kv_heads * a.head_tiles;
    int part = 0, each = INT32_MAX, seen, lo;
    if (a.parts == 0) {
      id = xcd_contiguous(id, a.sequences * units);
      sequence = index = id / units;
      unit = id - index * units;
      const Seen s = Seen::of(a, sequence);
      seen = __builtin_amdgcn_readfirstlane(s.seen);
      lo = __builtin_amdgcn_readfirstlane(s.lo);
    } else {
      const Cut cut(a, room);
      each = cut.each;
      if (id == 0) cut.note(a);
      none = id >= cut.all * units;
      if (none) return;
      id = xcd_contiguous(id, cut.all * units);
      index = id / units;
      unit = id - index * units;
      const uint64_t owner = __ballot(index >= cut.before && index < cut.before + cut.mine);
      int at = cut.before, found = 0, in = 0;
      for (int i = 0; i < cut.run; ++i) {
        const int s = (int)(threadIdx.x & 63) * cut.run + i, n = cut.parts_of(a, s);
        if (index >= at && index < at + n) found = s, in = index - at;
        at += n;
      }
      const int lane = __builtin_ctzll(owner);
      sequence = __builtin_amdgcn_readlane(found, lane);
      part = __builtin_amdgcn_readlane(in, lane);
      const Seen s = cut.run == 1 ? cut.only : Seen(a, cut.lengths[sequence]);
      seen = __builtin_amdgcn_readlane(s.seen, lane);
      lo = __builtin_amdgcn_readlane(s.lo, lane);
      count = (seen + each - 1) / each;
    }
    begin = lo + part * (a.parts > 0 ? each : 0);
    end = seen - part * (a.parts > 0 ? each : 0) <= each ? lo + seen : begin + each;
  }
};

// DIM: the head's elements, padded. A step: kStep positions. A row in LDS: kChunks of 16
// bytes, chunk c at place c ^ key_place (or value_place) of its row, so that lanes that
// read at the same time reach different banks.
template <class T, class S, int DIM>
struct Shape {
  static constexpr int kTiles = S::kBytes == 4 ? 1 : 2, kStep = 16 * kTiles;
  static constexpr int kElements = 16 / S::kBytes;       // of a chunk
  static constexpr int kChunks = DIM / kElements;        // of a row
  static constexpr int kOfLane = kChunks / 4;            // of a row, of a lane of the first product
  static constexpr int kRow = DIM * S::kBytes;
  static constexpr int kRows = 64 / kChunks;             // that one load instruction brings
  static constexpr int kLoads = kStep / kRows;           // of a step, of keys or of values
  static constexpr int kKeys = kStep * kRow, kSlot = 2 * kKeys;
  static constexpr int kDepth = kSlot >= kRing / 2 ? 2 : kRing / kSlot;  // steps in LDS
  static_assert(kChunks % 4 == 0 && kRows >= 1 && kRows <= 16 && 2 * kLoads < 64);
  // A lane reads a chunk of one of 16 neighbouring rows.
  __device__ static int key_place(int r) { return kChunks >= 8 ? r & 7 : (r ^ (r >> 2)) & 3; }
  // 16-bit: 32 bytes of each of four neighbouring rows. FP8: 16 of four and of the four 16 rows on. fp32: 64 of
  // each of four rows that are four apart.
  __device__ static int value_place(int r) {
    if constexpr (S::kBytes == 4) return ((r >> 2) & 3) << 2;
    if constexpr (S::kBytes == 2) return kChunks >= 16 ? (r & 3) << 1 : ((r >> 1) & 1) << 1;
    if constexpr (kChunks >= 16) return (r & 3) | ((r >> 4) & 1) << 2;
    return kChunks == 8 ? ((r >> 1) & 1) | ((r >> 4) & 1) << 1 : (r >> 4) & 1;
  }
};

// Four elements, eight or sixteen bytes, at any alignment.
template <class C>
__device__ inline void store4(const f32x4& v, char* p) {
  float f[C::VEC] = {};
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = v[i];
  const u32x4 w = C::pack(f);
  if constexpr (C::kBytes == 4) {
    *reinterpret_cast<u32x4_any*>(p) = w;
  } else {
    *reinterpret_cast<u32x2_any*>(p) = (u32x2){w[0], w[1]};
  }
}

// 16 bytes per lane from p to LDS at the named place + 16 x lane (see lds_place), as data that is
// read once: 13 % less time for 64 ragged sequences of up to 8192 positions.
__device__ inline void load_to_place_from(const char* p) {
  asm volatile("global_load_lds_dwordx4 %0, off nt" ::"v"(p) : "memory");
}

// FP8 values of element 16 f + col and eight positions, 4 g .. 4 g + 3 and 16 on: lanes 2 j
// and 2 j + 1 of 16 point at 16 codes of the j-th of eight rows, and lane i receives the
// eight rows' i-th codes.
template <class Sh>
__device__ inline u32x2 codes_at(LdsPtr from, int f, int g, int col) {
  using Lds2 = __attribute__((address_space(3))) i32x2*;
  const int j = col >> 1, r = (j >> 2) * 16 + 4 * g + (j & 3);
  const LdsPtr p = from + r * Sh::kRow + ((f ^ Sh::value_place(r)) << 4) + (col & 1) * 8;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32(reinterpret_cast<Lds2>(p)));
}

// WAVES: those of a workgroup, which share its positions and meet in LDS; more than one only where each sequence is
// one part.
template <class T, class S, int DIM, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 1) void paged_attention(AttentionArgs a) {
  using Sh = Shape<T, S, DIM>;
  constexpr int kTiles = Sh::kTiles, kStep = Sh::kStep, kOfLane = Sh::kOfLane, kFrags = S::kFragments;
  constexpr int kRow = Sh::kRow, kAll = 2 * Sh::kLoads;
  constexpr int kDepth = Sh::kDepth;
  constexpr int kOut = DIM / 16;
  static_assert(16 * DIM * 4 <= kDepth * Sh::kSlot && kMaxCut * 4 <= kDepth * Sh::kSlot);
  __shared__ __attribute__((aligned(1024))) char rings[WAVES][kDepth * Sh::kSlot];
  __shared__ __attribute__((aligned(16))) int founds[WAVES][kFound];

  const Part span(a, (int)blockIdx.x, reinterpret_cast<int*>(rings[0]));
  if (span.none) return;
  const int sequence = span.sequence, index = span.index, unit = span.unit;
  const int kv = unit / a.head_tiles, group = a.heads / a.kv_heads;
  const int head0 = unit % a.head_tiles * kHeads, heads = group - head0 < kHeads ? group - head0 : kHeads;

  const int wave = wave_of<WAVES>(), lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  char* const lds = rings[wave];
  int* const found = founds[wave];
  const int row_bytes = a.dim * S::kBytes;

  if (span.begin == span.end) {  // of a sequence that is one part; others have none then
    const int64_t first = (int64_t)sequence * a.heads + kv * group + head0;
    for (int e = (int)threadIdx.x * 4; e < heads * a.dim; e += 256 * WAVES) {
      store4<typename T::Codec>((f32x4){0.0f, 0.0f, 0.0f, 0.0f}, a.out + (first * a.dim + e) * T::kBytes);
    }
    if ((int)threadIdx.x < heads && a.lse != nullptr) a.lse[first + threadIdx.x] = -__builtin_inff();
    return;
  }
  int begin = span.begin, end = span.end;
  if constexpr (WAVES > 1) {
    const int each = ((end - begin + WAVES - 1) / WAVES + kStep - 1) / kStep * kStep;
    begin += wave * each;
    end = end - begin < each ? end : begin + each;  // no more than begin: nothing for this wave
  }

  // The columns' queries: of each chunk of a row the elements that this lane has.
  u32x4 q[kOfLane][kFrags];
  {
    const int h = kv * group + head0 + (col < heads ? col : 0);
    const char* from = a.q + ((int64_t)sequence * a.q_token + (int64_t)h * a.q_head) * T::kBytes;
#pragma unroll
    for (int s = 0; s < kOfLane; ++s) {
#pragma unroll
      for (int f = 0; f < kFrags; ++f) {
        const int e = (4 * s + g) * Sh::kElements + f * (16 / T::kBytes);
        q[s][f] = (u32x4){0u, 0u, 0u, 0u};
        if (e < a.dim) q[s][f] = *reinterpret_cast<const u32x4_any*>(from + e * T::kBytes);
      }
    }
  }

  // Slots of the positions from `first` on, kFound of them; -1 for none.
  const int64_t* table = a.table + (int64_t)sequence * a.table_width;
  auto find = [&](int first, auto each) __attribute__((always_inline)) {
    constexpr int kEach = decltype(each)::value;  // of a lane
    int64_t page[kEach];
    int in_page[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int t = first + i * 64 + lane, last = end - 1;
      const uint32_t u = (uint32_t)(t < last ? t : last);
      const uint32_t at = (uint32_t)(((uint64_t)u * a.page_magic) >> a.page_shift);
      page[i] = table[at];
      in_page[i] = (int)(u - at * (uint32_t)a.page);
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const bool there = first + i * 64 + lane < end && page[i] >= 0 && page[i] < a.pages;
      found[i * 64 + lane] = there ? (int)page[i] * a.page + in_page[i] : -1;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  };
  auto look = [&](int first) __attribute__((always_inline)) {
    if (end - first <= 64) {
      find(first, IntC<1>{});
    } else {
      find(first, IntC<kFound / 64>{});
    }
  };
  // The lane's row and chunk of a load instruction's kRows rows.
  const int load_row = lane / Sh::kChunks, load_chunk = lane % Sh::kChunks;
  const int64_t slot_bytes = (int64_t)a.kv_heads * row_bytes;
  const char *const keys = a.keys + (int64_t)kv * row_bytes, *const values = a.values + (int64_t)kv * row_bytes;
  // Asks for a step of keys and values; which of its positions there are.
  auto ask = [&](int first, LdsPtr to) __attribute__((always_inline)) {
    const int at = first - begin;
    if (at > 0 && at % kFound == 0) look(first);
    const int mine = found[at % kFound + (lane & (kStep - 1))];
#pragma unroll
    for (int i = 0; i < Sh::kLoads; ++i) {
      const int r = i * Sh::kRows + load_row;
      const int slot = found[at % kFound + r];
      // past the row its last chunk will do, and for a position that is not there any row
      const int key_byte = (load_chunk ^ Sh::key_place(r)) * 16, value_byte = (load_chunk ^ Sh::value_place(r)) * 16;
      const int64_t row = (int64_t)(uint32_t)(slot < 0 ? 0 : slot) * slot_bytes;
      lds_place(to + i * 1024);
      place_ready();
      load_to_place_from(keys + (row + (key_byte < row_bytes ? key_byte : row_bytes - 16)));
      lds_place(to + Sh::kKeys + i * 1024);
      place_ready();
      load_to_place_from(values + (row + (value_byte < row_bytes ? value_byte : row_bytes - 16)));
    }
    return (uint32_t)__ballot(mine >= 0);
  };

  f32x4 out[kOut] = {};
  // P is taken by base: top - kLift, or 0 while there is none.
  float top = -__builtin_inff(), base = 0.0f, sum = 0.0f;
  // An infinite value makes NaN of what it should not where P has a low part (zero, or of the other sign) or is zero in
  // 16 bits, and large ones of bfloat16 and float32 make an infinite sum of finite values. So where a wave has a sum
  // that is not finite, it takes all its steps again, AGAIN, one at a time: infinite values count for themselves, by 1
  // where their P is a normal float32, and P is scaled down. Codes of FP8 are not large. The look at the sums costs
  // 0.1 us a call; all steps again as much as the call (64 sequences of up to 8192 positions, bf16: 201 us, with a NaN in
  // every page 381).
  constexpr int kLiftAgain = S::kBytes == 1 ? T::kLift : T::kLiftAgain;
  auto step = [&](const LdsPtr slot, uint32_t seen, auto again) __attribute__((always_inline)) {
    constexpr bool AGAIN = decltype(again)::value;
    constexpr int kLift = AGAIN ? kLiftAgain : T::kLift;
    constexpr uint32_t kEvery = kStep == 32 ? 0xffffffffu : 0xffffu;
    const bool all = (seen & kEvery) == kEvery;
    u32x4 k[kTiles][kOfLane];
#pragma unroll
    for (int s = 0; s < kOfLane; ++s) {
#pragma unroll
      for (int j = 0; j < kTiles; ++j) {
        k[j][s] = lds_load<u32x4>(slot + (16 * j + col) * kRow + (((4 * s + g) ^ Sh::key_place(col)) << 4));
      }
    }
    if (row_bytes < kRow) {  // there is more in LDS than the row
#pragma unroll
      for (int s = 0; s < kOfLane; ++s) {
#pragma unroll
        for (int j = 0; j < kTiles; ++j) {
          if ((4 * s + g) * 16 >= row_bytes) k[j][s] = (u32x4){0u, 0u, 0u, 0u};
        }
      }
    }
    f32x4 score[kTiles] = {};
#pragma unroll
    for (int s = 0; s < kOfLane; ++s) {
#pragma unroll
      for (int j = 0; j < kTiles; ++j) {
        u32x4 f[kFrags];
        S::fragments(k[j][s], f);
#pragma unroll
        for (int i = 0; i < kFrags; ++i) score[j] = T::mma(f[i], q[s][i], score[j]);
      }
    }
    const LdsPtr from = slot + Sh::kKeys;
    if (!all) {  // values that are not seen may be anything: zeros
      const u32x4 zeros = {0u, 0u, 0u, 0u};
      for (int i = 0; i < Sh::kLoads; ++i) {
        if (!(seen >> (i * Sh::kRows + load_row) & 1)) lds_store(zeros, from + i * 1024 + lane * 16);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
    float most = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < kTiles; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x = score[j][i] * a.score_scale;
        if (!all && !(seen >> (16 * j + 4 * g + i) & 1)) x = -__builtin_inff();
        score[j][i] = x;
        most = __builtin_fmaxf(most, x);
      }
    }
    if (__any(most > top + kSlack)) {
      most = __builtin_fmaxf(most, __shfl_xor(most, 16));
      most = __builtin_fmaxf(most, __shfl_xor(most, 32));
      const float now = __builtin_fmaxf(top, most);
      const float keep = __builtin_amdgcn_exp2f(top - (now == -__builtin_inff() ? 0.0f : now));
      base = now == -__builtin_inff() ? 0.0f : now - kLift;
      top = now;
      sum *= keep;
#pragma unroll
      for (int f = 0; f < kOut; ++f) out[f] *= keep;
    }
    f32x4 ones[kTiles];
#pragma unroll
    for (int j = 0; j < kTiles; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (AGAIN) ones[j][i] = score[j][i] - base + kLift >= -126.0f ? 1.0f : 0.0f;
        score[j][i] = __builtin_amdgcn_exp2f(score[j][i] - base);
        sum += score[j][i];
      }
    }
    // Elements past the head's are computed with what is in LDS there, and not stored.
    if constexpr (T::kBytes == 2) {
      u32x4 high, low, one;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if constexpr (AGAIN) one[2 * j + i] = T::pack(ones[j][2 * i], ones[j][2 * i + 1]);
          const float x = score[j][2 * i], y = score[j][2 * i + 1];
          const uint32_t h = T::pack(x, y);
          high[2 * j + i] = h;
          low[2 * j + i] = T::pack(x - T::low(h), y - T::high(h));
        }
      }
#pragma unroll
      for (int f = 0; f < kOut; ++f) {
        u32x4 w;
        if constexpr (S::kBytes == 2) {
          // Four rows of 16 elements, turned over: row 4 g + col / 4 of a tile, and 16 on, which has the same place.
          using Lds4 = __attribute__((address_space(3))) s16x4*;
          const int r = 4 * g + (col >> 2), c = (2 * f + ((col >> 1) & 1)) ^ Sh::value_place(r);
          const LdsPtr p = from + r * kRow + c * 16 + (col & 1) * 8;
          const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<Lds4>(p)));
          const u32x2 y =
              __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<Lds4>(p + 16 * kRow)));
          w = (u32x4){x[0], x[1], y[0], y[1]};
        } else {
          uint32_t e[2], e2[2];
          const u32x2 x = codes_at<Sh>(from, f, g, col);
          S::four(x[0], e);
          S::four(x[1], e2);
          w = (u32x4){e[0], e[1], e2[0], e2[1]};
        }
        if constexpr (AGAIN) {
          const u32x4 rest = not_finite<T>(w);
          out[f] = T::mma(rest, one, out[f]);
          w ^= rest;
        }
        out[f] = T::mma(w, high, out[f]);
        out[f] = T::mma(w, low, out[f]);
      }
    } else {
      auto add = [&](f32x4& o, u32x4 w, int j) __attribute__((always_inline)) {
        if constexpr (AGAIN) {
          const u32x4 rest = not_finite<T>(w);
          o = T::mma(rest, __builtin_bit_cast(u32x4, ones[j]), o);
          w ^= rest;
        }
        o = T::mma(w, __builtin_bit_cast(u32x4, score[j]), o);
      };
#pragma unroll
      for (int f = 0; f < kOut; ++f) {
        if constexpr (S::kBytes == 4) {
          u32x4 w;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = 4 * g + i, c = (4 * f + (col >> 2)) ^ Sh::value_place(r);
            w[i] = lds_load<uint32_t>(from + r * kRow + c * 16 + (col & 3) * 4);
          }
          add(out[f], w, 0);
        } else {
          const u32x2 x = codes_at<Sh>(from, f, g, col);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            uint32_t e[4];
            S::four(x[j], e);
            add(out[f], (u32x4){e[0], e[1], e[2], e[3]}, j);
          }
        }
      }
    }
  };

  const LdsPtr slots = (LdsPtr)lds;
  int lift = T::kLift;
  if (WAVES == 1 || begin < end) {
    uint32_t seen[kDepth] = {};
    look(begin);
    // The queries are here, as the slots are: a wait of the compiler's inside the loop would be one for the steps on
    // their way too.
#pragma unroll
    for (int s = 0; s < kOfLane; ++s) {
#pragma unroll
      for (int f = 0; f < kFrags; ++f) asm volatile("" : "+v"(q[s][f]));
    }
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      if (begin + d * kStep < end) seen[d] = ask(begin + d * kStep, slots + d * Sh::kSlot);
    }
    for (int first = begin; first < end; first += kDepth * kStep) {
#pragma unroll
      for (int d = 0; d < kDepth; ++d) {
        const int now = first + d * kStep;
        if (now < end) {
          if (now + (kDepth - 1) * kStep < end) {
            loads_landed<(kDepth - 1) * kAll>();
          } else {
            loads_landed();
          }
          step(slots + d * Sh::kSlot, seen[d], std::false_type{});
          if (now + kDepth * kStep < end) {
            lds_read();
            seen[d] = ask(now + kDepth * kStep, slots + d * Sh::kSlot);
          }
        }
      }
    }
    if (__builtin_expect(__any(!finite(out)), 0)) {
      lift = kLiftAgain;
      top = -__builtin_inff();
      base = sum = 0.0f;
#pragma unroll
      for (int f = 0; f < kOut; ++f) out[f] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
      look(begin);
      for (int first = begin; first < end; first += kStep) {
        lds_read();
        const uint32_t here = ask(first, slots);
        loads_landed();
        step(slots, here, std::true_type{});
      }
    }
  }
  sum += __shfl_xor(sum, 16);
  sum += __shfl_xor(sum, 32);
  top -= lift;  // the sums' power of two from here on

  if constexpr (WAVES > 1) {
    // As join_parts, of the waves.
    float* const sums = reinterpret_cast<float*>(lds);
    if (col < heads) {
#pragma unroll
      for (int f = 0; f < kOut; ++f) *reinterpret_cast<f32x4*>(sums + col * DIM + 16 * f + 4 * g) = out[f];
    }
    if (g == 0) *reinterpret_cast<f32x2*>(found + 2 * col) = (f32x2){top, sum};
    __syncthreads();
    const int quads = a.dim / 4;
    for (int i = threadIdx.x; i < heads * quads; i += 64 * WAVES) {
      const int h = i / quads, quad = i - h * quads;
      f32x2 stats[WAVES];
      float all_top = -__builtin_inff(), total = 0.0f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        stats[w] = *reinterpret_cast<const f32x2*>(founds[w] + 2 * h);
        all_top = __builtin_fmaxf(all_top, stats[w][0]);
      }
      const float all_base = all_top == -__builtin_inff() ? 0.0f : all_top;
      f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
      auto part = [&](int w) __attribute__((always_inline)) {
        return *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(rings[w]) + h * DIM + 4 * quad);
      };
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        const float p = __builtin_amdgcn_exp2f(stats[w][0] - all_base);
        o += p * part(w);
        total += p * stats[w][1];
      }
      if (__builtin_expect(S::kBytes > 1 && !finite(o), 0)) {
        o = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
        total = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) add_down(o, total, part(w), stats[w], all_base);
        all_top = all_base - kDown;
      }
      const int64_t head = (int64_t)sequence * a.heads + kv * group + head0 + h;
      const float inverse = total == 0.0f ? 0.0f : a.value_scale / total;
      o = total == 0.0f ? (f32x4){0.0f, 0.0f, 0.0f, 0.0f} : o * inverse;
      store4<typename T::Codec>(o, a.out + (head * a.dim + 4 * quad) * T::kBytes);
      if (quad == 0 && a.lse != nullptr) {
        a.lse[head] = total == 0.0f ? -__builtin_inff() : (all_top + __builtin_log2f(total)) * kLn2;
      }
    }
    return;
  }
  if (col >= heads) return;
  const int in_sequence = kv * group + head0 + col;
  const int64_t head = (int64_t)sequence * a.heads + in_sequence;
  if (span.count > 1) {
    const int64_t at = (int64_t)index * a.heads + in_sequence;
#pragma unroll
    for (int f = 0; f < kOut; ++f) {
      if (16 * f < a.dim) *reinterpret_cast<f32x4*>(a.partial + at * a.dim + 16 * f + 4 * g) = out[f];
    }
    if (g == 0) {
      float* const stats = stats_of(a) + at * 2;
      stats[0] = top;
      stats[1] = sum;
    }
  } else {
    const float inverse = sum == 0.0f ? 0.0f : a.value_scale / sum;
#pragma unroll
    for (int f = 0; f < kOut; ++f) {
      if (16 * f < a.dim) {
        const f32x4 o = sum == 0.0f ? (f32x4){0.0f, 0.0f, 0.0f, 0.0f} : out[f] * inverse;
        store4<typename T::Codec>(o, a.out + (head * a.dim + 16 * f + 4 * g) * T::kBytes);
      }
    }
    if (g == 0 && a.lse != nullptr) {
      a.lse[head] = sum == 0.0f ? -__builtin_inff() : (top + __builtin_log2f(sum)) * kLn2;
    }
  }
}

constexpr int64_t kMaxPositions = int64_t(1) << 30;  // of a sequence: a step past the last is still an int
constexpr int64_t kMaxBlocks = (int64_t(1) << 24) - 1;

// The sums of a sequence's parts, a head a workgroup. A thread has four elements of every
// `lanes`-th part, and takes kAhead parts at a time.
template <class C, int THREADS>
__global__ __launch_bounds__(THREADS) void join_parts(AttentionArgs a) {
  __shared__ f32x4 sums[THREADS];
  __shared__ f32x2 tops[THREADS];
  constexpr int kAhead = THREADS == 64 ? 4 : 8;
  const int sequence = (int)(blockIdx.x / a.heads), head = (int)(blockIdx.x - sequence * a.heads);
  const int* const notes = notes_of(a) + 2 * sequence;
  const int first = notes[0], count = notes[1], tid = threadIdx.x;
  if (count == 1) return;  // its wave stored the result
  const int quads = a.dim / 4, lanes = THREADS / quads, quad = tid % quads, of = tid / quads;
  const float* const from = a.partial + ((int64_t)first * a.heads + head) * a.dim + quad * 4;
  const f32x2* const stats = reinterpret_cast<const f32x2*>(stats_of(a)) + (int64_t)first * a.heads + head;
  const int64_t stride = (int64_t)a.heads * a.dim;
  f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  float top = -__builtin_inff(), total = 0.0f;
  const bool large = a.value_scale == 1.0f;  // values may be: not those of an FP8 cache
  if (of < lanes) {
    for (int p0 = of; p0 < count; p0 += kAhead * lanes) {
      f32x4 part[kAhead];
      f32x2 stat[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int p = p0 + i * lanes, at = p < count ? p : p0;
        part[i] = *reinterpret_cast<const f32x4*>(from + at * stride);
        stat[i] = stats[(int64_t)at * a.heads];
        if (p >= count) stat[i] = (f32x2){-__builtin_inff(), 0.0f};
      }
      const float before = top;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) top = __builtin_fmaxf(top, stat[i][0]);
      const float base = top == -__builtin_inff() ? 0.0f : top, keep = __builtin_amdgcn_exp2f(before - base);
      o *= keep;
      total *= keep;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const float w = __builtin_amdgcn_exp2f(stat[i][0] - base);
        if (p0 + i * lanes < count) o += w * part[i];
        total += w * stat[i][1];
      }
    }
    if (__builtin_expect(large && !finite(o), 0)) {
      const float base = top == -__builtin_inff() ? 0.0f : top;
      o = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
      total = 0.0f;
      for (int p = of; p < count; p += lanes) {
        add_down(o, total, *reinterpret_cast<const f32x4*>(from + p * stride), stats[(int64_t)p * a.heads], base);
      }
      top = base - kDown;
    }
  }
  sums[tid] = o;
  tops[tid] = (f32x2){top, total};
  __syncthreads();
  if (tid >= quads) return;
  float all_top = top;
  for (int i = 1; i < lanes; ++i) all_top = __builtin_fmaxf(all_top, tops[i * quads + tid][0]);
  const float base = all_top == -__builtin_inff() ? 0.0f : all_top;
  o = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
  total = 0.0f;
  for (int i = 0; i < lanes; ++i) {
    const float w = __builtin_amdgcn_exp2f(tops[i * quads + tid][0] - base);
    o += w * sums[i * quads + tid];
    total += w * tops[i * quads + tid][1];
  }
  if (__builtin_expect(large && !finite(o), 0)) {
    o = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    total = 0.0f;
    for (int i = 0; i < lanes; ++i) add_down(o, total, sums[i * quads + tid], tops[i * quads + tid], base);
    all_top = base - kDown;
  }
  const float inverse = total == 0.0f ? 0.0f : a.value_scale / total;
  o = total == 0.0f ? (f32x4){0.0f, 0.0f, 0.0f, 0.0f} : o * inverse;
  store4<C>(o, a.out + ((int64_t)blockIdx.x * a.dim + tid * 4) * C::kBytes);
  if (tid == 0 && a.lse != nullptr) {
    a.lse[blockIdx.x] = total == 0.0f ? -__builtin_inff() : (all_top + __builtin_log2f(total)) * kLn2;
  }
}

int64_t bytes_of(int32_t dtype) { return dtype == kF32 ? 4 : dtype == kF16 || dtype == kBF16 ? 2 : 1; }

int head_tiles_of(int64_t heads, int64_t kv_heads) { return (int)((heads / kv_heads + kHeads - 1) / kHeads); }

// Bytes of LDS of a step's keys and values.
int64_t step_bytes(int64_t dim, int64_t cache_bytes) {
  return (cache_bytes == 4 ? 16 : 32) * (dim <= 64 ? 64 : dim <= 128 ? 128 : 256) * cache_bytes * 2;
}

// Parts of all sequences together, at most, or 0 where each is one. Few sequences: as many as fill the LDS of the 256
// CUs, all of one length. More of them end in parts that are shorter and leave CUs to wait, so then there are several
// for each place; each costs about what kPartCost positions do, and the sum of both is least for a square root. The
// host takes half of the positions that the table has room for, the workgroups what there are: then many of the grid's
// find nothing to do, so it is limited. bf16, 8 heads of 128, ragged, us, this and 8 parts a sequence: 64 of up to 8192
// 191, 193; 128 of up to 4096 192, 205; 32 of up to 4096 55, 57; 64 of up to 1000 in tables for 131072 32, 36; 128 in
// tables for 32768 57, 67. It loses with 64 of up to 32768: 729, 712.
constexpr double kPartCost = 150;
// Workgroups of a key-value head that fit the card.
int64_t places_of(int64_t units, int64_t dim, int64_t cache_bytes) {
  const int64_t two = 2 * step_bytes(dim, cache_bytes);
  const int64_t slots = 256 * (160 * 1024 / ((two > kRing ? two : kRing) + kFound * 4));
  return (slots + units - 1) / units;
}
bool few(int64_t sequences, int64_t places) { return 4 * sequences <= places; }
int64_t parts_of(int64_t sequences, int64_t units, int64_t positions, int64_t dim, int64_t cache_bytes) {
  if (positions <= kMinPart || sequences > kMaxCut) return 0;
  const int64_t places = places_of(units, dim, cache_bytes);
  int64_t parts = places;
  if (!few(sequences, places)) {
    const double half = 0.5 * (double)(sequences * positions);  // lengths differ
    const int64_t more = (int64_t)__builtin_sqrt(half * (double)places / kPartCost);
    parts = sequences + (more < 4 * places ? more : 4 * places);
    parts = parts > places ? parts : places;
    parts = parts > 2 * sequences ? parts : 2 * sequences;
  }
  const int64_t most = sequences * ((positions + kMinPart - 1) / kMinPart) + sequences;  // of the shortest parts
  parts = parts < most ? parts : most;
  return parts * units <= kMaxBlocks ? parts : 0;  // so many heads fill the card by themselves
}

// Who takes a sequence of a key-value head: a wave, the waves of a workgroup, or parts of it are shared out. Without
// parts there is no second launch, and no length but its own to read, but where one sequence is much longer than the
// others its waves are waited for: a step costs a wave 1 us alone.
// A wave, for steps that are few for the number of them (B workgroups). bf16, 8 heads of 128, ragged, up to so many
// positions, us, a wave, waves and parts: B 8192: 64 42, 117, 231; 512 182, 228, 362. B 2048: 64 12, 30, 32; 512 53, 62,
// 65; 1024 106, 99, 110. B 512: 64 6.6, 8.6, 9.9; 256 12.7, 12.3, 13.6; 512 20.9, 18.8, 20.9.
// Waves, for contexts that they are through with soon; the more work there is beside it, the longer. Us, waves and
// parts: B 8: 256 6.8, 9.6; 768 10.2, 11.2; 1024 12.4, 11.2. B 64: 512 9.0, 10.9; 1024 15.2, 12.3. B 256: 1024 17.1,
// 20.0; 2048 30.9, 31.1. B 1024: 1024 55, 61; 2048 99, 103. B 2048: 2048 183, 198.
enum Way { kWave, kWaves, kParts };
Way way_of(int64_t blocks, int64_t seen, int64_t dim, int64_t cache_bytes) {
  const int64_t bytes = step_bytes(dim, cache_bytes), each = cache_bytes == 4 ? 16 : 32;
  const int64_t steps = (seen + each - 1) / each;
  if (steps <= 2 || steps <= blocks / 128) return kWave;
  const int64_t waves = 2 * bytes > kRing ? 2 : 4;
  const int64_t soon = blocks < 128 ? 6 : blocks < 1024 ? 8 : 16;  // of a wave, of 16 KB or less
  return steps <= waves * (bytes > kRing / 2 ? soon / 2 : soon) ? kWaves : kParts;
}

template <class T, class S, int DIM>
void run_waves(const AttentionArgs& a, int64_t blocks, bool whole, hipStream_t st) {
  using Sh = Shape<T, S, DIM>;
  constexpr int kWaves = Sh::kDepth * Sh::kSlot > kRing ? 2 : 4;  // rings that fit a CU's LDS
  if (whole) {
    paged_attention<T, S, DIM, kWaves><<<(unsigned)blocks, 64 * kWaves, 0, st>>>(a);
  } else {
    paged_attention<T, S, DIM, 1><<<(unsigned)blocks, 64, 0, st>>>(a);
  }
}

template <class T, class S>
int32_t run_dim(const AttentionArgs& a, int64_t blocks, bool whole, hipStream_t st) {
  if (a.dim <= 64) {
    run_waves<T, S, 64>(a, blocks, whole, st);
  } else if (a.dim <= 128) {
    run_waves<T, S, 128>(a, blocks, whole, st);
  } else {
    run_waves<T, S, 256>(a, blocks, whole, st);
  }
  int32_t status = launch_status();
  if (status == 0 && a.parts > 0) {
    // Few parts a sequence on average: a wave for each head (64 sequences of up to 8 parts: 5 us less).
    const unsigned grid = (unsigned)(a.sequences * a.heads);
    if (a.parts <= 16 * (int64_t)a.sequences) {
      join_parts<typename T::Codec, 64><<<grid, 64, 0, st>>>(a);
    } else {
      join_parts<typename T::Codec, 512><<<grid, 512, 0, st>>>(a);
    }
    status = launch_status();
  }
  return status;
}

template <class T>
int32_t run_cache(const AttentionArgs& a, int64_t blocks, bool whole, int32_t cache_dtype, hipStream_t st) {
  if (cache_dtype == kF8E4M3) return run_dim<T, FromCodes<T, kF8E4M3>>(a, blocks, whole, st);
  if (cache_dtype == kF8E5M2) return run_dim<T, FromCodes<T, kF8E5M2>>(a, blocks, whole, st);
  return run_dim<T, AsIs<T>>(a, blocks, whole, st);
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
                                                 int64_t head_dim, int64_t page_size, int64_t table_width,
                                                 int32_t cache_dtype) {
  if (sequences <= 0 || !attention_sizes_ok(sequences, n_q_heads, n_kv_heads, head_dim, page_size, table_width)) return 0;
  const int64_t units = n_kv_heads * head_tiles_of(n_q_heads, n_kv_heads);
  const int64_t positions = page_size * table_width, bytes = bytes_of(cache_dtype);
  // With a window fewer positions are seen, which never makes parts of what is none without.
  if (way_of(sequences * units, positions, head_dim, bytes) != kParts) return 0;
  const int64_t parts = parts_of(sequences, units, positions, head_dim, bytes);
  return parts == 0 ? 0 : parts * n_q_heads * (head_dim + 2) * 4 + sequences * 8;
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
      pages > INT32_MAX / page_size) {
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
  const int64_t units = n_kv_heads * a.head_tiles;
  const int64_t positions = page_size * table_width, seen = a.window > 0 && a.window < positions ? a.window : positions;
  a.parts = (int)parts_of(sequences, units, positions, head_dim, bytes_of(cache_dtype));
  const Way way = way_of(sequences * units, seen, head_dim, bytes_of(cache_dtype));
  if (way != kParts) a.parts = 0;
  const int64_t places = places_of(units, head_dim, bytes_of(cache_dtype));
  a.part_cost = few(sequences, places) ? 0.0f : (float)(kPartCost / (double)places);
  const bool whole = way != kWave && a.parts == 0;
  if (a.parts > 0 && (workspace == nullptr || !host_aligned(workspace, 16))) return (int32_t)hipErrorInvalidValue;
  // t / page for t < 2^31: t * magic >> shift, magic = floor(2^(31 + bits) / page) + 1 with
  // 2^bits >= page. What magic is too large by, at most 1, adds less than 2^-bits <= 1 / page.
  int bits = 0;
  while ((int64_t(1) << bits) < page_size) ++bits;
  a.page_shift = 31 + bits;
  a.page_magic = (uint32_t)(((unsigned __int128)1 << (31 + bits)) / (uint64_t)page_size + 1);
  a.score_scale = scale * key_scale * kLog2e;
  a.value_scale = value_scale;
  const int64_t blocks = (a.parts > 0 ? a.parts : sequences) * units;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case kF32: return run_cache<F32>(a, blocks, whole, cache_dtype, st);
    case kF16: return run_cache<F16>(a, blocks, whole, cache_dtype, st);
    default: return run_cache<Bf16>(a, blocks, whole, cache_dtype, st);
  }
}

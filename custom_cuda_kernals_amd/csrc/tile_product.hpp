// Tiled matrix products on the CDNA4 matrix cores, for groups of ragged size.
//
//   D[p][q] = sum_c P(p, c) * Q(q, c)
//
// P and Q are read as rows (the contracted index c contiguous) or as columns
// (p or q contiguous, a row of memory per c). A workgroup of WP x WQ waves owns
// a tile of D; each wave holds FP x FQ fragments of 16 x 16 in registers. The
// contraction goes in steps of 128 bytes a row (64 16-bit, 32 fp32 or 256 4-bit
// elements); a step's tiles of P and Q wait in LDS, two steps deep:
//
//   half 1 of step t:  read the second half's fragments | multiply the first's
//   barrier: step t + 1 has landed, and step t has been read
//   half 2 of step t:  read step t + 1's first fragments, ask for step t + 2 |
//                      multiply the second half's
//
// so global loads have a whole step, and LDS reads half a step, of products in
// front of them. The MFMA takes Q's fragment as its first operand, so a lane
// holds consecutive q of one p and stores whole vectors.
#pragma once

#include "launch.hpp"

namespace cck {

using bf16x8 = __bf16 __attribute__((ext_vector_type(8)));
using f16x8 = _Float16 __attribute__((ext_vector_type(8)));
using s16x4 = short __attribute__((ext_vector_type(4)));
using i32x8 = int __attribute__((ext_vector_type(8)));

constexpr int kRowBytes = 128;          // bytes of a row in one step
constexpr int kChunks = kRowBytes / 16;  // 16-byte chunks of them
// Steps are addressed by 32-bit byte offsets from a 64-bit base that moves with
// the tile and the step: at most 256 rows of this many bytes.
constexpr int64_t kMaxRowLength = int64_t(1) << 22;

// ---------------------------------------------------------------------------
// Element types. A fragment is what one lane holds for one MFMA step of 64
// bytes a row: lane l has row l % 16 and a 16-byte chunk (l / 16 of the half step's
// four; 4-bit: 2 (l / 16) + half of the step's eight).
// ---------------------------------------------------------------------------

struct ElemBF16 {
  static constexpr int kBytes = 2;
  static constexpr bool kScaled = false;
  template <int KS>
  __device__ static f32x4 mma(const u32x4& q, const u32x4& p, const f32x4& c, int, int) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, q), __builtin_bit_cast(bf16x8, p), c, 0,
                                                   0, 0);
  }
};
struct ElemF16 {
  static constexpr int kBytes = 2;
  static constexpr bool kScaled = false;
  template <int KS>
  __device__ static f32x4 mma(const u32x4& q, const u32x4& p, const f32x4& c, int, int) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, q), __builtin_bit_cast(f16x8, p), c, 0, 0,
                                                  0);
  }
};
// Four MFMAs of depth 4: MFMA j takes element j of every lane's chunk.
struct ElemF32 {
  static constexpr int kBytes = 4;
  static constexpr bool kScaled = false;
  template <int KS>
  __device__ static f32x4 mma(const u32x4& q, const u32x4& p, f32x4 c, int, int) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(bits_f32(q[j]), bits_f32(p[j]), c, 0, 0, 0);
    }
    return c;
  }
};

// OCP MXFP4: e2m1 codes, two a byte, with an E8M0 scale for each chunk of 32.
// Rows are counted in bytes of codes. A lane's two chunks of a step are
// neighbours, so that one 16-bit read brings both their scales: byte KS of the
// scale operand is that of half KS.
struct ElemFP4 {
  static constexpr int kBytes = 1;
  static constexpr bool kScaled = true;
  template <int KS>
  __device__ static f32x4 mma(const u32x4& q, const u32x4& p, const f32x4& c, int q_scale, int p_scale) {
    constexpr int kFp4 = 4;  // the operand format e2m1
    const i32x8 a = {(int)q[0], (int)q[1], (int)q[2], (int)q[3], 0, 0, 0, 0};
    const i32x8 b = {(int)p[0], (int)p[1], (int)p[2], (int)p[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, kFp4, kFp4, KS, q_scale, KS, p_scale);
  }
};

// ---------------------------------------------------------------------------
// Groups: offsets[e] .. offsets[e + 1] are the rows of group e. Whatever the
// offsets hold, the rows a kernel touches lie in [0, rows).
// ---------------------------------------------------------------------------

constexpr int kMaxGroups = 1024;

__device__ inline int64_t clamp_row(int64_t v, int64_t rows) { return v < 0 ? 0 : v > rows ? rows : v; }

// One tile of the rows: rows [row, row + count) of group `group`; group < 0 for
// the rows before the first and behind the last group, which are zeros in the
// output; count == 0 for a tile past the last one.
struct RowTileAt {
  int64_t row;
  int count, group;
};

// The number of row tiles of BP rows, and which rows the tile `index` of them
// holds. Threads hold the groups' tile counts, whose prefix sums say where each
// group's tiles begin. The pseudo groups 0 (rows before the first group) and
// groups + 1 (behind the last) take part. Every thread of the workgroup calls.
// Where the offsets decrease somewhere, groups overlap or miss rows, but every
// tile still lies in [0, rows), and there are no more of them than the grid has.
template <int BP, int THREADS>
struct RowTiles {
  static constexpr int kPer = (kMaxGroups + 2 + THREADS - 1) / THREADS;
  int first[kPer];  // tiles before this thread's groups
  int64_t lo[kPer];
  int n[kPer];
  int total;

  // slots: THREADS / 64 ints; found: 2 words. `most`: tiles that the grid has room for.
  __device__ RowTiles(const int64_t* offsets, int groups, int64_t rows, int most, int* slots, int64_t* found) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (tid < 2) found[tid] = 0;
    const int per = (groups + 2 + THREADS - 1) / THREADS;
    int sum = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = tid * per + i;
      lo[i] = 0;
      n[i] = 0;
      if (i < per && e < groups + 2) {
        lo[i] = e == 0 ? 0 : clamp_row(offsets[e - 1], rows);
        const int64_t hi = e == groups + 1 ? rows : clamp_row(offsets[e], rows);
        n[i] = hi > lo[i] ? (int)(hi - lo[i]) : 0;
      }
      first[i] = sum;
      sum += (n[i] + BP - 1) / BP;
    }
    int before = sum;  // inclusive prefix over the wave
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int v = __shfl_up(before, d);
      if (lane >= d) before += v;
    }
    if (lane == 63) slots[wave] = before;
    __syncthreads();
    int base = before - sum;
    total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
      const int v = slots[w];
      if (w < wave) base += v;
      total += v;
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) first[i] += base;
    total = total < 0 || total > most ? most : total;
  }

  __device__ RowTileAt at(int index, int groups, int64_t* found) const {
    const int tid = threadIdx.x;
    const int per = (groups + 2 + THREADS - 1) / THREADS;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int k = index - first[i];
      if (k >= 0 && k < (n[i] + BP - 1) / BP) {
        const int e = tid * per + i;
        found[0] = lo[i] + (int64_t)k * BP;
        found[1] = ((int64_t)(n[i] - k * BP < BP ? n[i] - k * BP : BP) << 32) | (uint32_t)(e == groups + 1 ? 0 : e);
      }
    }
    __syncthreads();
    const int64_t row = found[0], w = found[1];
    RowTileAt t;
    t.row = row_uniform(row);
    t.count = __builtin_amdgcn_readfirstlane((int)(w >> 32));
    t.group = __builtin_amdgcn_readfirstlane((int)(uint32_t)w) - 1;
    return t;
  }

  __device__ static int64_t row_uniform(int64_t v) {
    const uint32_t a = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v);
    const uint32_t b = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(v >> 32));
    return (int64_t)((uint64_t)b << 32 | a);
  }
};

// Workgroups go to the 8 XCDs in turn; this numbering gives each XCD one run of
// consecutive tiles, whose operands then meet in its L2.
__device__ inline int xcd_contiguous(int id, int total) {
  const int xcd = id & 7, k = id >> 3, each = total >> 3, rest = total & 7;
  return xcd * each + (xcd < rest ? xcd : rest) + k;
}

// Tiles in blocks of kBlockP row tiles, in each block the row tiles of one
// column tile after another: what runs at the same time on an XCD shares rows
// of P and of Q.
constexpr int kBlockP = 8;
__device__ inline void tile_order(int t, int tiles_p, int tiles_q, int* tp, int* tq) {
  const int block = t / (kBlockP * tiles_q), p0 = block * kBlockP;
  const int height = tiles_p - p0 < kBlockP ? tiles_p - p0 : kBlockP;
  const int r = t - block * kBlockP * tiles_q;
  *tq = r / height;
  *tp = p0 + r % height;
}

// ---------------------------------------------------------------------------
// Operand tiles in LDS.
// ---------------------------------------------------------------------------

using LdsPtr = __attribute__((address_space(3))) char*;

// The buffer resource of everything from `base` (the same in every lane) on.
__device__ inline u32x4 buffer_from(const char* base) {
  const uint64_t b = (uint64_t)base;
  return (u32x4){(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)b),
                 (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(b >> 32)), 0x7fffffffu, (uint32_t)kBufDword3};
}
constexpr uint32_t kOutOfRange = 0x80000000u;  // an offset past the end of every buffer: reads as zeros

// 16 bytes per lane from `off` on to LDS at `to` + 16 x lane, without registers
// in between. Written out because the compiler, which does not know that the two
// halves of the LDS tiles are apart, would wait for these loads before every
// later LDS read; their one wait is loads_landed.
__device__ inline void load_to_lds(const u32x4& buffer, uint32_t off, LdsPtr to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)to)), "v"(off), "s"(buffer)
               : "memory");
}
__device__ inline void load_to_lds4(const u32x4& buffer, uint32_t off, LdsPtr to) {  // 4 bytes per lane
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds"
               :
               : "s"(__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)to)), "v"(off), "s"(buffer)
               : "memory");
}
__device__ inline void loads_landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// 16 bytes from p, of which the first `bytes` (0 .. 16) are in range; the others
// are zeros. BYTES: of an element.
template <int BYTES>
__device__ inline u32x4 load_part(const char* p, int bytes) {
  if (bytes >= 16) return *reinterpret_cast<const u32x4_any*>(p);
  u32x4 v = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int i = 0; i < 16 / BYTES; ++i) {
    if (i * BYTES < bytes) {
      uint32_t e;
      if constexpr (BYTES == 4) e = *reinterpret_cast<const u32_any*>(p + i * 4);
      if constexpr (BYTES == 2) e = *reinterpret_cast<const u16_any*>(p + i * 2);
      if constexpr (BYTES == 1) e = (uint8_t)p[i];
      v[i * BYTES / 4] |= e << (8 * (i * BYTES % 4));
    }
  }
  return v;
}

// An operand of R rows whose contracted index is contiguous. In LDS a row is
// 128 bytes; its chunk c sits at position c ^ swizzle(row), so that the 8 lanes
// that read one chunk of 8 rows reach different banks. PERM: fragment f of a
// block of 64 rows holds rows 16 (i / 4) + 4 f + i % 4 (i: the lane's row of 16)
// in place of 16 f + i, so that a lane's results of four fragments are 16
// consecutive rows.
template <class T, int R, int NW, bool PERM>
struct RowOperand {
  static constexpr int kLds = R * kRowBytes;
  static constexpr int kLoads = R * kChunks / (NW * 64);
  static_assert(kLoads * NW * 64 == R * kChunks);
  __device__ static int swizzle(int row) { return PERM ? (row & 3) | ((row >> 4) & 1) << 2 : row & 7; }
  __device__ static int frag_row(int f, int i) {
    return PERM ? (f >> 2) * 64 + 16 * (i >> 2) + 4 * (f & 3) + (i & 3) : 16 * f + i;
  }

  const char* base;  // the tile's first row at the current step
  int64_t ld;        // bytes
  int rows, left;    // rows in range; bytes of a row still in range

  __device__ RowOperand(const void* p, int64_t ld_bytes, int rows_, int64_t length)
      : base(static_cast<const char*>(p)), ld(ld_bytes), rows(rows_), left((int)(length * T::kBytes)) {}
  __device__ void advance() {
    base += kRowBytes;
    left -= kRowBytes;
  }
  // Load i of the thread: its row, and the chunk that goes to its position.
  __device__ static int load_row(int i) { return (i * NW * 64 + (int)threadIdx.x) / kChunks; }
  __device__ static int load_chunk(int i) { return ((int)threadIdx.x & (kChunks - 1)) ^ swizzle(load_row(i)); }

  // Straight into LDS: chunks in range are whole, and aligned.
  __device__ void fetch(LdsPtr lds) const {
    const u32x4 r = buffer_from(base);
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int row = load_row(i), at = load_chunk(i) * 16;
      // Past the last row any row will do; past the row's end zeros, from an offset out of range.
      const uint32_t off = at < left ? (uint32_t)(row < rows ? row : rows - 1) * (uint32_t)ld + at : kOutOfRange;
      load_to_lds(r, off, lds + (i * NW + wave) * 1024);
    }
  }
  // Through registers: any alignment and length.
  __device__ void load(u32x4 (&v)[kLoads]) const {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int row = load_row(i), at = load_chunk(i) * 16;
      const int part = left - at < 0 ? 0 : left - at;
      v[i] = load_part<T::kBytes>(base + (int64_t)(row < rows ? row : rows - 1) * ld + (part ? at : 0), part);
    }
  }
  __device__ static void store(const u32x4 (&v)[kLoads], LdsPtr lds) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      *reinterpret_cast<__attribute__((address_space(3))) u32x4*>(lds + (i * NW * 64 + (int)threadIdx.x) * 16) = v[i];
    }
  }
  // Fragment f of the wave whose rows begin at row0, half ks of the step.
  __device__ static u32x4 fragment(LdsPtr lds, int row0, int f, int ks) {
    const int lane = threadIdx.x & 63, row = row0 + frag_row(f, lane & 15), g = lane >> 4;
    const int at = row * kRowBytes + (((T::kScaled ? 2 * g + ks : ks * 4 + g) ^ swizzle(row)) * 16);
    return *reinterpret_cast<__attribute__((address_space(3))) u32x4*>(lds + at);
  }
};

// An operand whose R rows are contiguous for one contracted index: a step is
// kDepth rows of memory, R elements of each. In LDS a chunk sits at position
// chunk ^ swizzle(c). 16-bit fragments are transposed by ds_read_b64_tr_b16
// (lanes 4 j .. 4 j + 3 of 16 point at 16 elements of the j-th of four rows, and
// lane i receives the four rows' i-th elements); fp32 ones are read one by one.
template <class T, int R, int NW>
struct ColOperand {
  static constexpr int kDepth = kRowBytes / T::kBytes;
  static constexpr int kWide = R * T::kBytes / 16;  // chunks of a row in LDS
  static constexpr int kLds = R * kRowBytes;
  static constexpr int kLoads = R * kChunks / (NW * 64);
  static_assert(kLoads * NW * 64 == R * kChunks);
  __device__ static int swizzle(int c) { return T::kBytes == 2 ? (c & 3) * 2 : ((c >> 2) & 3) * 4; }
  __device__ static int frag_row(int f, int i) { return 16 * f + i; }

  const char* base;  // the tile's first column at the current step
  int64_t ld;        // bytes
  int wide;          // bytes in range of a row of memory
  int64_t left;      // contracted rows in range

  __device__ ColOperand(const void* p, int64_t ld_bytes, int rows, int64_t length)
      : base(static_cast<const char*>(p)), ld(ld_bytes), wide(rows * T::kBytes), left(length) {}
  __device__ void advance() {
    base += kDepth * ld;
    left -= kDepth;
  }
  __device__ static int load_c(int i) { return (i * NW * 64 + (int)threadIdx.x) / kWide; }
  __device__ static int load_chunk(int i) { return ((int)threadIdx.x & (kWide - 1)) ^ swizzle(load_c(i)); }

  __device__ void fetch(LdsPtr lds) const {
    const u32x4 r = buffer_from(base);
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int c = load_c(i), at = load_chunk(i) * 16;
      const uint32_t off = c < left && at < wide ? (uint32_t)c * (uint32_t)ld + at : kOutOfRange;
      load_to_lds(r, off, lds + (i * NW + wave) * 1024);
    }
  }
  __device__ void load(u32x4 (&v)[kLoads]) const {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int c = load_c(i), at = load_chunk(i) * 16;
      const int part = c < left && at < wide ? wide - at : 0;
      v[i] = load_part<T::kBytes>(part ? base + (int64_t)c * ld + at : base, part);
    }
  }
  __device__ static void store(const u32x4 (&v)[kLoads], LdsPtr lds) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      *reinterpret_cast<__attribute__((address_space(3))) u32x4*>(lds + (i * NW * 64 + (int)threadIdx.x) * 16) = v[i];
    }
  }
  __device__ static u32x4 fragment(LdsPtr lds, int row0, int f, int ks) {
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    if constexpr (T::kBytes == 2) {
      const int col = row0 + 16 * f + 4 * (i & 3), c0 = ks * 32 + g * 8 + (i >> 2);
      const int chunk = (col >> 3) ^ swizzle(c0);  // c0 + 4 swizzles alike
      const LdsPtr p = lds + (c0 * kWide + chunk) * 16 + (col & 4) * 2;
      using Lds4 = __attribute__((address_space(3))) s16x4*;
      const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<Lds4>(p)));
      const u32x2 b =
          __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<Lds4>(p + 4 * kWide * 16)));
      return (u32x4){a[0], a[1], b[0], b[1]};
    } else {
      const int col = row0 + 16 * f + i, c0 = ks * 16 + g * 4;
      const LdsPtr p = lds + (c0 * kWide + ((col >> 2) ^ swizzle(c0))) * 16 + (col & 3) * 4;
      u32x4 v;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[j] = *reinterpret_cast<__attribute__((address_space(3))) uint32_t*>(p + j * kWide * 16);
      }
      return v;
    }
  }
};

// The E8M0 scales of an operand of R rows (`blocks` bytes a row): eight bytes a
// row and step in LDS. PERM as in RowOperand.
template <class Operand, int R, int NW>
struct Scales {
  static constexpr int kLds = R * kChunks;
  static constexpr int kLoads = (R * 2 + NW * 64 - 1) / (NW * 64);  // of four scales
  const char* base;
  int64_t ld;
  int rows, left;

  __device__ Scales(const void* p, int64_t blocks, int rows_)
      : base(static_cast<const char*>(p)), ld(blocks), rows(rows_), left((int)blocks) {}
  __device__ void advance() {
    base += kChunks;
    left -= kChunks;
  }
  __device__ void fetch(LdsPtr lds) const {
    const u32x4 r = buffer_from(base);
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int d = i * NW * 64 + (int)threadIdx.x, row = d >> 1, at = (d & 1) * 4;
      if ((i + 1) * NW * 64 <= R * 2 || (i * NW + wave) * 64 < R * 2) {
        const uint32_t off = at < left ? (uint32_t)(row < rows ? row : rows - 1) * (uint32_t)ld + at : kOutOfRange;
        load_to_lds4(r, off, lds + (i * NW + wave) * 256);
      }
    }
  }
  __device__ void load(uint32_t (&v)[kLoads]) const {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int d = i * NW * 64 + (int)threadIdx.x, row = d >> 1, at = (d & 1) * 4;
      const char* p = base + (int64_t)(row < rows ? row : rows - 1) * ld + at;
      v[i] = 0u;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (at + j < left) v[i] |= (uint32_t)(uint8_t)p[j] << (8 * j);
      }
    }
  }
  __device__ static void store(const uint32_t (&v)[kLoads], LdsPtr lds) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int d = i * NW * 64 + (int)threadIdx.x;
      if ((i + 1) * NW * 64 <= R * 2 || d < R * 2) *reinterpret_cast<__attribute__((address_space(3))) uint32_t*>(lds + d * 4) = v[i];
    }
  }
  // Both halves' scales of the lane's row of fragment f.
  __device__ static int fragment(LdsPtr lds, int row0, int f) {
    const int lane = threadIdx.x & 63, row = row0 + Operand::frag_row(f, lane & 15);
    return *reinterpret_cast<__attribute__((address_space(3))) uint16_t*>(lds + row * kChunks + 2 * (lane >> 4));
  }
};

// In place of the scales of the types that have none.
struct NoScales {
  static constexpr int kLds = 0, kLoads = 1;
  __device__ void advance() {}
  __device__ void fetch(LdsPtr) const {}
  __device__ void load(uint32_t (&)[1]) const {}
  __device__ static void store(const uint32_t (&)[1], LdsPtr) {}
  __device__ static int fragment(LdsPtr, int, int) { return 0; }
};

// ---------------------------------------------------------------------------
// The product.
// ---------------------------------------------------------------------------

template <class T, class P, class Q, class PS, class QS, int WP, int WQ, int FP, int FQ, bool DIRECT>
struct Product {
  // P, Q, the scales of P and of Q.
  static constexpr int kAtQ = P::kLds, kAtPS = kAtQ + Q::kLds, kAtQS = kAtPS + PS::kLds, kStage = kAtQS + QS::kLds;

  // acc[fp][fq] += the product over `steps` steps. lds0, lds1: kStage bytes each.
  __device__ static void run(P p, Q q, PS ps, QS qs, int steps, LdsPtr lds0, LdsPtr lds1, f32x4 (&acc)[FP][FQ]) {
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int p0 = (wave / WQ) * FP * 16, q0 = (wave % WQ) * FQ * 16;
    u32x4 pa[FP], qa[FQ], pb[FP], qb[FQ];  // the fragments of the first and second half
    int sp[FP] = {}, sq[FQ] = {};          // and the scales of both
    u32x4 pv[DIRECT ? 1 : P::kLoads], qv[DIRECT ? 1 : Q::kLoads];
    uint32_t psv[DIRECT ? 1 : PS::kLoads], qsv[DIRECT ? 1 : QS::kLoads];

    auto ask = [&](LdsPtr lds) {  // the next step's loads on their way
      if constexpr (DIRECT) {
        p.fetch(lds);
        q.fetch(lds + kAtQ);
        ps.fetch(lds + kAtPS);
        qs.fetch(lds + kAtQS);
      } else {
        p.load(pv);
        q.load(qv);
        ps.load(psv);
        qs.load(qsv);
      }
      p.advance();
      q.advance();
      ps.advance();
      qs.advance();
    };
    auto put = [&](LdsPtr lds) {  // and in LDS
      if constexpr (!DIRECT) {
        P::store(pv, lds);
        Q::store(qv, lds + kAtQ);
        PS::store(psv, lds + kAtPS);
        QS::store(qsv, lds + kAtQS);
      }
    };
    auto landed = [&] {
      if constexpr (DIRECT) loads_landed();
      __syncthreads();
    };
    auto read = [&](LdsPtr lds, int ks, u32x4 (&pf)[FP], u32x4 (&qf)[FQ]) {
#pragma unroll
      for (int f = 0; f < FQ; ++f) qf[f] = Q::fragment(lds + kAtQ, q0, f, ks);
#pragma unroll
      for (int f = 0; f < FP; ++f) pf[f] = P::fragment(lds, p0, f, ks);
    };
    auto read_scales = [&](LdsPtr lds) {
      if constexpr (T::kScaled) {
#pragma unroll
        for (int f = 0; f < FQ; ++f) sq[f] = QS::fragment(lds + kAtQS, q0, f);
#pragma unroll
        for (int f = 0; f < FP; ++f) sp[f] = PS::fragment(lds + kAtPS, p0, f);
      }
    };
    auto multiply = [&](auto half, const u32x4 (&pf)[FP], const u32x4 (&qf)[FQ]) {
#pragma unroll
      for (int a = 0; a < FP; ++a) {
#pragma unroll
        for (int b = 0; b < FQ; ++b) acc[a][b] = T::template mma<decltype(half)::value>(qf[b], pf[a], acc[a][b], sq[b], sp[a]);
      }
    };
    auto step = [&](LdsPtr now, LdsPtr next) {
      read(now, 1, pb, qb);
      read_scales(now);
      multiply(IntC<0>{}, pa, qa);
      put(next);
      landed();
      read(next, 0, pa, qa);
      ask(now);
      multiply(IntC<1>{}, pb, qb);
    };

    // Steps past the last are asked for and read too, as zeros (nothing of them is
    // in range), so that the loop has no conditions; their products are left out.
    if (steps <= 0) return;
    ask(lds0);
    put(lds0);
    landed();
    read(lds0, 0, pa, qa);
    ask(lds1);
    int t = 0;
    for (; t + 2 <= steps; t += 2) {
      step(lds0, lds1);
      step(lds1, lds0);
    }
    if (t < steps) {
      read(lds0, 1, pb, qb);
      read_scales(lds0);
      multiply(IntC<0>{}, pa, qa);
      multiply(IntC<1>{}, pb, qb);
    }
    if constexpr (DIRECT) loads_landed();
  }
};

// Stores a wave's fragments: rows [p0, rows) of `out` (row stride ld elements),
// columns [q0, cols). VEC: the rows' vectors are aligned.
template <class C, bool PERM, int FP, int FQ>
__device__ inline void store_tile(const f32x4 (&acc)[FP][FQ], char* out, int64_t ld, int p0, int q0, int rows, int cols,
                                  bool aligned) {
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
#pragma unroll
  for (int a = 0; a < FP; ++a) {
    const int p = p0 + 16 * a + i;
    if (p >= rows) continue;
    char* const row = out + (int64_t)p * ld * C::kBytes;
    constexpr int kRun = PERM ? 16 : 4;  // consecutive columns of a lane
#pragma unroll
    for (int b = 0; b < FQ; b += kRun / 4) {
      const int q = q0 + (PERM ? (b >> 2) * 64 + 16 * g : 16 * b + 4 * g);
      float f[kRun];
#pragma unroll
      for (int j = 0; j < kRun; ++j) f[j] = acc[a][b + j / 4][j % 4];
      if (aligned && q + kRun <= cols) {
        if constexpr (kRun * C::kBytes >= 16) {
#pragma unroll
          for (int v = 0; v < kRun / C::VEC; ++v) {
            float part[C::VEC];
#pragma unroll
            for (int j = 0; j < C::VEC; ++j) part[j] = f[v * C::VEC + j];
            *reinterpret_cast<u32x4*>(row + (int64_t)(q + v * C::VEC) * C::kBytes) = C::pack(part);
          }
        } else {
          const float part[8] = {f[0], f[1], f[2], f[3], 0.0f, 0.0f, 0.0f, 0.0f};
          const u32x4 w = C::pack(part);
          *reinterpret_cast<u32x2*>(row + (int64_t)q * C::kBytes) = (u32x2){w[0], w[1]};
        }
      } else {
#pragma unroll
        for (int j = 0; j < kRun; ++j) {
          if (q + j < cols) C::store1(row, q + j, f[j]);
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Rows against the weights of their group: out[s][:] = x[s] * w[e]^T (QROWS: w[e]
// is [cols][length]) or x[s] * w[e] (w[e] is [length][cols]). Rows of no group are
// zeros. offsets == nullptr: one group of all rows.
// ---------------------------------------------------------------------------

struct RowsArgs {
  const char *x, *w, *x_scale, *w_scale;
  const int64_t* offsets;
  char* out;
  int64_t rows, length;  // elements of T
  int groups, cols, tiles_q, most;
};

// Two waves on a SIMD (256 registers a lane); tiles that go through registers need more.
template <class T, class C, bool QROWS, int WP, int WQ, int FP, int FQ, bool DIRECT>
__global__ __launch_bounds__(WP* WQ * 64, DIRECT ? 2 : 1) void rows_product(RowsArgs a) {
  constexpr int BP = WP * FP * 16, BQ = WQ * FQ * 16, NW = WP * WQ, kDepth = kRowBytes / T::kBytes;
  using P = RowOperand<T, BP, NW, false>;
  using Q = std::conditional_t<QROWS, RowOperand<T, BQ, NW, true>, ColOperand<T, BQ, NW>>;
  using PS = std::conditional_t<T::kScaled, Scales<P, BP, NW>, NoScales>;
  using QS = std::conditional_t<T::kScaled, Scales<Q, BQ, NW>, NoScales>;
  using Prod = Product<T, P, Q, PS, QS, WP, WQ, FP, FQ, DIRECT>;
  __shared__ __attribute__((aligned(1024))) char lds0[Prod::kStage];
  __shared__ __attribute__((aligned(1024))) char lds1[Prod::kStage];
  __shared__ int slots[NW];
  __shared__ int64_t found[2];

  RowTileAt at;
  int tp, tq;
  if (a.offsets != nullptr) {
    const RowTiles<BP, NW * 64> tiles(a.offsets, a.groups, a.rows, a.most, slots, found);
    const int total = tiles.total * a.tiles_q;
    if ((int)blockIdx.x >= total) return;
    tile_order(xcd_contiguous(blockIdx.x, total), tiles.total, a.tiles_q, &tp, &tq);
    at = tiles.at(tp, a.groups, found);
    if (at.count == 0) return;
  } else {
    tile_order(xcd_contiguous(blockIdx.x, gridDim.x), a.most, a.tiles_q, &tp, &tq);
    at.row = (int64_t)tp * BP;
    at.count = a.rows - at.row < BP ? (int)(a.rows - at.row) : BP;
    at.group = 0;
  }

  const int col = tq * BQ, width = a.cols - col < BQ ? a.cols - col : BQ;
  const int64_t e = at.group < 0 ? 0 : at.group;
  const int64_t ldp = a.length * T::kBytes, ldq = QROWS ? ldp : (int64_t)a.cols * T::kBytes;
  const char* wt = a.w + e * a.length * a.cols * T::kBytes + (QROWS ? col * ldq : (int64_t)col * T::kBytes);
  f32x4 acc[FP][FQ] = {};
  const int steps = at.group < 0 ? 0 : (int)((a.length + kDepth - 1) / kDepth);
  const P p(a.x + at.row * ldp, ldp, at.count, a.length);
  const Q q(wt, ldq, width, a.length);
  if constexpr (T::kScaled) {
    const int64_t blocks = a.length / 16;
    Prod::run(p, q, PS(a.x_scale + at.row * blocks, blocks, at.count),
              QS(a.w_scale + (e * a.cols + col) * blocks, blocks, width), steps, (LdsPtr)lds0, (LdsPtr)lds1, acc);
  } else {
    Prod::run(p, q, PS(), QS(), steps, (LdsPtr)lds0, (LdsPtr)lds1, acc);
  }

  const int wave = threadIdx.x >> 6;
  const bool aligned = a.cols % C::VEC == 0 && aligned16(a.out);
  store_tile<C, QROWS>(acc, a.out + (at.row * a.cols + col) * C::kBytes, a.cols, (wave / WQ) * FP * 16,
                       (wave % WQ) * FQ * 16, at.count, width, aligned);
}

constexpr int64_t kMaxThreads = int64_t(1) << 32;  // of one launch

template <class T, class C, bool QROWS, int WP, int WQ, int FP, int FQ, bool DIRECT>
int32_t launch_rows(RowsArgs a, hipStream_t st) {
  constexpr int BP = WP * FP * 16, BQ = WQ * FQ * 16, kThreads = WP * WQ * 64;
  const int64_t edges = a.offsets == nullptr ? 1 : a.groups + 2;  // each group ends inside one tile at most
  int64_t most = (a.rows + edges * (BP - 1)) / BP;
  most = most < a.rows ? most : a.rows;
  const int64_t tiles_q = ((int64_t)a.cols + BQ - 1) / BQ;
  if (most * tiles_q * kThreads >= kMaxThreads) return (int32_t)hipErrorInvalidValue;
  a.most = (int)most;
  a.tiles_q = (int)tiles_q;
  rows_product<T, C, QROWS, WP, WQ, FP, FQ, DIRECT><<<(unsigned)(most * tiles_q), kThreads, 0, st>>>(a);
  return launch_status();
}

// Sizes every kernel here accepts: 32-bit row counts and columns, rows that 32-bit
// offsets reach from a tile's base.
inline bool sizes_ok(int64_t rows, int64_t groups, int64_t n_bytes, int64_t k_bytes) {
  return rows >= 0 && rows <= INT32_MAX && groups >= 1 && groups <= kMaxGroups && n_bytes <= kMaxRowLength &&
         k_bytes <= kMaxRowLength;
}

}  // namespace cck

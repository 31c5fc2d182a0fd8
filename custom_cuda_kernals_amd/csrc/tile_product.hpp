// Tiled matrix products on the CDNA4 matrix cores, for groups of ragged size.
//
//   D[p][q] = sum_c P(p, c) * Q(q, c)
//
// P and Q are read as rows (the contracted index c contiguous) or as columns
// (p or q contiguous, a row of memory per c). A workgroup of WP x WQ waves owns
// a tile of D; each wave holds FP x FQ fragments of 16 x 16 in registers. The
// contraction goes in steps of 128 bytes a row (64 16-bit, 32 fp32 or 256 4-bit
// elements), two MFMAs deep (eight for fp32). Two steps' tiles of P and Q are in LDS:
//
//   half 1 of step t:  multiply the first 64 bytes' fragments | read the others';
//                      barrier: step t has been read; ask for step t + 2
//   barrier: step t + 1 has landed
//   half 2 of step t:  multiply them | read step t + 1's first; ask for step t + 2
//
// so a load has a step and more of products in front of it, and an LDS read half a
// step. Reads and loads are issued between the products, and the loads evenly: at once
// they would hold each other up, with the matrix cores idle. The MFMA takes Q's
// fragment as its first operand, so a lane holds consecutive q of one p and stores
// whole vectors.
#pragma once

#include "launch.hpp"

namespace cck {

using bf16x8 = __bf16 __attribute__((ext_vector_type(8)));
using f16x8 = _Float16 __attribute__((ext_vector_type(8)));
using s16x4 = short __attribute__((ext_vector_type(4)));
using i32x8 = int __attribute__((ext_vector_type(8)));

constexpr int kHalf = 64;  // bytes of a row in one MFMA step
// Loads are addressed by 32-bit byte offsets from a 64-bit base that moves with the
// tile and the step: at most 256 rows of this many bytes.
constexpr int64_t kMaxRowLength = int64_t(1) << 22;

// ---------------------------------------------------------------------------
// Element types. A fragment is what one lane holds for one MFMA step of 64
// bytes a row: lane l has row l % 16 and the 16-byte chunk l / 16.
// ---------------------------------------------------------------------------

// Products into the accumulation registers (mma_acc). Left to the compiler, 64
// accumulators a lane do not stay there: it moves them to the other registers and back
// around every product. The compiler does not see that these are matrix instructions, so
// the wait states that they need are written out: two behind a vector instruction that
// writes an operand (operands_ready), 18 before the sums are read (acc_ready). That no copy
// of the compiler's is nearer is tested on the built code (tests/test_matrix_asm_cpu.py).
__device__ inline void operands_ready() { asm volatile("s_nop 1"); }
template <int N>
__device__ inline void computed_here(int (&v)[N]) {  // and not behind the wait
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(v[i]));
}
template <int FP, int FQ>
__device__ inline void acc_ready(f32x4 (&acc)[FP][FQ]) {
  asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7" ::: "memory");
#pragma unroll
  for (int a = 0; a < FP; ++a) {
#pragma unroll
    for (int b = 0; b < FQ; ++b) asm volatile("" : "+a"(acc[a][b]));
  }
}

struct ElemBF16 {
  static constexpr bool kAccumulates = true;  // has mma_acc
  __device__ static void mma_acc(const u32x4& q, const u32x4& p, f32x4& c, int, int) {
    asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(q), "v"(p));
  }
  static constexpr int kFold = 0;
  static constexpr int kBytes = 2;
  static constexpr bool kScaled = false;
  __device__ static f32x4 mma(const u32x4& q, const u32x4& p, const f32x4& c, int, int) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, q), __builtin_bit_cast(bf16x8, p), c, 0,
                                                   0, 0);
  }
};
struct ElemF16 {
  static constexpr bool kAccumulates = true;
  __device__ static void mma_acc(const u32x4& q, const u32x4& p, f32x4& c, int, int) {
    asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(q), "v"(p));
  }
  static constexpr int kFold = 0;
  static constexpr int kBytes = 2;
  static constexpr bool kScaled = false;
  __device__ static f32x4 mma(const u32x4& q, const u32x4& p, const f32x4& c, int, int) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, q), __builtin_bit_cast(f16x8, p), c, 0, 0,
                                                  0);
  }
};
// Four MFMAs of depth 4: MFMA j takes element j of every lane's chunk. Sums are folded
// every 16 halves of steps (256 elements) into a second accumulator, so that their rounding
// errors do not grow with the whole length.
struct ElemF32 {
  static constexpr bool kAccumulates = false;
  static constexpr int kFold = 16;
  static constexpr int kBytes = 4;
  static constexpr bool kScaled = false;
  __device__ static f32x4 mma(const u32x4& q, const u32x4& p, f32x4 c, int, int) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(bits_f32(q[j]), bits_f32(p[j]), c, 0, 0, 0);
    }
    return c;
  }
};

// OCP MXFP4: e2m1 codes, two a byte, with an E8M0 scale for each chunk of 32, in
// the low byte of the scale operand. Rows are counted in bytes of codes.
struct ElemFP4 {
  static constexpr bool kAccumulates = true;
  __device__ static void mma_acc(const u32x4& q, const u32x4& p, f32x4& c, int q_scale, int p_scale) {
    asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0] cbsz:4 blgp:4"
                 : "+a"(c)
                 : "v"(q), "v"(p), "v"(q_scale), "v"(p_scale));
  }
  static constexpr int kFold = 0;
  static constexpr int kBytes = 1;
  static constexpr bool kScaled = true;
  __device__ static f32x4 mma(const u32x4& q, const u32x4& p, const f32x4& c, int q_scale, int p_scale) {
    constexpr int kFp4 = 4;  // the operand format e2m1
    const i32x8 a = {(int)q[0], (int)q[1], (int)q[2], (int)q[3], 0, 0, 0, 0};
    const i32x8 b = {(int)p[0], (int)p[1], (int)p[2], (int)p[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, kFp4, kFp4, 0, q_scale, 0, p_scale);
  }
};

// ---------------------------------------------------------------------------
// Groups: offsets[e] .. offsets[e + 1] are the rows of group e. Whatever the
// offsets hold, the rows a kernel touches lie in [0, rows).
// ---------------------------------------------------------------------------

constexpr int kMaxGroups = 1024;

// A value that all lanes hold, to the scalar registers.
__device__ inline int64_t uniform(int64_t v) {
  const uint32_t a = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v);
  const uint32_t b = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(v >> 32));
  return (int64_t)((uint64_t)b << 32 | a);
}

__device__ inline int64_t clamp_row(int64_t v, int64_t rows) { return v < 0 ? 0 : v > rows ? rows : v; }

// One tile of the rows: rows [row, row + count) of group `group`; group < 0 for
// the rows before the first and behind the last group, which are zeros in the
// output; count == 0 for a tile past the last one.
struct RowTileAt {
  int64_t row;
  int count, group;
};

// The number of row tiles of BP rows, and which rows the tile `index` of them holds.
// A thread has a run of groups, and knows how many tiles come before them. The pseudo
// groups 0 (rows before the first group) and groups + 1 (behind the last) take part. Every
// thread of the workgroup calls. Where the offsets decrease somewhere, groups overlap or
// miss rows, but every tile still lies in [0, rows), and there are no more of them than
// the grid has room for.
template <int BP, int THREADS>
struct RowTiles {
  struct Shared {
    int bound[kMaxGroups + 1];  // the offsets, in [0, rows]
    int sums[THREADS / 64];     // tiles of each wave's groups
    int found[3];               // a tile: its first row, its rows, its group
  };
  Shared& in;
  int groups, rows, per, first, total;

  // `most`: tiles that the grid has room for.
  __device__ RowTiles(Shared& shared, const int64_t* offsets, int groups_, int64_t rows_, int most)
      : in(shared), groups(groups_), rows((int)rows_), per((groups_ + 1 + THREADS) / THREADS) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int e = tid; e <= groups; e += THREADS) in.bound[e] = (int)clamp_row(offsets[e], rows);
    if (tid < 3) in.found[tid] = 0;  // for a tile past the last one
    __syncthreads();
    int sum = 0;
    for (int i = 0; i < per; ++i) sum += tiles_of(height(tid * per + i));
    int before = sum;  // inclusive prefix over the wave
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int v = __shfl_up(before, d);
      if (lane >= d) before += v;
    }
    if (lane == 63) in.sums[wave] = before;
    __syncthreads();
    first = before - sum;
    total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
      const int v = in.sums[w];
      if (w < wave) first += v;
      total += v;
    }
    total = __builtin_amdgcn_readfirstlane(total < 0 || total > most ? most : total);
  }
  __device__ int begin(int e) const { return e == 0 ? 0 : in.bound[e - 1]; }
  __device__ int height(int e) const {
    if (e > groups + 1) return 0;
    const int n = (e == groups + 1 ? rows : in.bound[e]) - begin(e);
    return n > 0 ? n : 0;
  }
  __device__ static int tiles_of(int n) { return (int)(((uint32_t)n + BP - 1) / BP); }

  __device__ RowTileAt at(int index) const {
    int before = first;
    for (int i = 0; i < per; ++i) {
      const int e = (int)threadIdx.x * per + i, n = height(e), k = index - before;
      before += tiles_of(n);
      if (k >= 0 && index < before) {
        in.found[0] = begin(e) + k * BP;
        in.found[1] = n - k * BP < BP ? n - k * BP : BP;
        in.found[2] = e == groups + 1 ? 0 : e;
      }
    }
    __syncthreads();
    RowTileAt t;
    t.row = __builtin_amdgcn_readfirstlane(in.found[0]);
    // Offsets in no order can name a tile twice: still none of it past the last row.
    const int count = __builtin_amdgcn_readfirstlane(in.found[1]), left = rows - (int)t.row;
    t.count = count < left ? count : left;
    t.group = __builtin_amdgcn_readfirstlane(in.found[2]) - 1;
    return t;
  }
};

// Workgroups go to the 8 XCDs in turn; this numbering gives each XCD one run of
// consecutive tiles, whose operands then meet in its L2.
__device__ inline int xcd_contiguous(int id, int total) {
  const int xcd = id & 7, k = id >> 3, each = total >> 3, rest = total & 7;
  return xcd * each + (xcd < rest ? xcd : rest) + k;
}

// Tiles in blocks of HEIGHT row tiles, in each block the row tiles of one column tile
// after another: what runs at the same time on an XCD shares rows of P and of Q.
template <int HEIGHT = 8>
__device__ inline void tile_order(int t, int tiles_p, int tiles_q, int* tp, int* tq) {
  const int block = t / (HEIGHT * tiles_q), p0 = block * HEIGHT;
  const int height = tiles_p - p0 < HEIGHT ? tiles_p - p0 : HEIGHT;
  const int r = t - block * HEIGHT * tiles_q;
  *tq = r / height;
  *tp = p0 + r % height;
}

// ---------------------------------------------------------------------------
// Operand tiles in LDS.
// ---------------------------------------------------------------------------

using LdsPtr = __attribute__((address_space(3))) char*;

// A pointer that is the same in all lanes, in the scalar registers.
__device__ inline const char* in_scalars(const char* p) {
  asm("" : "+s"(p));
  return p;
}
// The buffer resource of everything from `base` on, the same in every lane.
__device__ inline u32x4 buffer_from(const char* base) {
  const uint64_t b = (uint64_t)base;
  return (u32x4){(uint32_t)b, (uint32_t)(b >> 32), 0x7fffffffu, (uint32_t)kBufDword3};
}
constexpr uint32_t kOutOfRange = 0x80000000u;  // an offset past the end of every buffer

// BYTES (16 or 4) per lane from `off` on to LDS at `to` + BYTES x lane, without registers
// in between. ONCE: as data that nobody reads again. Written out because the compiler,
// which does not know that the slots of a ring are apart, would wait for these loads
// before every later LDS read; their one wait is loads_landed (all but the last LEFT
// of the wave's loads).
// In two instructions, the first naming the place (register M0, which the compiler reserves
// and does not use by itself): one other instruction at least belongs between them.
__device__ inline void lds_place(LdsPtr to) {
  asm volatile("s_mov_b32 m0, %0" ::"s"(__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)to)) : "memory");
}
template <int BYTES, bool ONCE>
__device__ inline void load_to_place(const u32x4& buffer, uint32_t off) {
  if constexpr (BYTES == 4) {
    asm volatile("buffer_load_dword %0, %1, 0 offen lds" ::"v"(off), "s"(buffer) : "memory");
  } else if constexpr (ONCE) {
    asm volatile("buffer_load_dwordx4 %0, %1, 0 offen nt lds" ::"v"(off), "s"(buffer) : "memory");
  } else {
    asm volatile("buffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(off), "s"(buffer) : "memory");
  }
}
__device__ inline void place_ready() { asm volatile("s_nop 0" ::: "memory"); }
template <int LEFT = 0>
__device__ inline void loads_landed() {
  static_assert(LEFT < 64);
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LEFT) : "memory");
}
// The wave's LDS reads have their values.
__device__ inline void lds_read() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
// The workgroup's waves meet; loads that are on their way stay so, unlike at __syncthreads.
__device__ inline void meet() { asm volatile("s_barrier" ::: "memory"); }

// w without its first `bytes`, zeros behind the rest (none left from 16 on).
__device__ inline u32x4 drop_bytes(u32x4 w, int bytes) {
  if (bytes & 8) w = (u32x4){w[2], w[3], 0u, 0u};
  if (bytes & 4) w = (u32x4){w[1], w[2], w[3], 0u};
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = __builtin_amdgcn_alignbyte(i < 3 ? w[i + 1] : 0u, w[i], (uint32_t)bytes & 3u);
  if (bytes >= 16) r = (u32x4){0u, 0u, 0u, 0u};
  return r;
}
// The sixteen bytes at `at` of a row that ends at `end`, or the row's last sixteen
// where those reach over its end (at, end: from p on; rows have 16 bytes or more, and
// may begin before p); what drop_bytes(.., over_end(at, end)) then makes right.
__device__ inline u32x4 load_before_end(const char* p, int at, int end) {
  return *reinterpret_cast<const u32x4_any*>(p + (at < end - 16 ? at : end - 16));
}
__device__ inline int over_end(int at, int end) { return at < end - 16 ? 0 : at - (end - 16); }

// Thread and wave among the NW waves that share a tile.
template <int NW>
__device__ inline int thread_of() {
  return (int)threadIdx.x & (NW * 64 - 1);
}
template <int NW>
__device__ inline int wave_of() {
  return __builtin_amdgcn_readfirstlane(thread_of<NW>() >> 6);
}

// A value that is kept in a register, and not computed again at each use.
__device__ inline int in_vector(int v) {
  asm("" : "+v"(v));
  return v;
}
template <class V>
__device__ inline V lds_load(LdsPtr p) {
  return *reinterpret_cast<__attribute__((address_space(3))) V*>(p);
}
template <class V>
__device__ inline void lds_store(const V& v, LdsPtr p) {
  *reinterpret_cast<__attribute__((address_space(3))) V*>(p) = v;
}

// An operand of R rows whose contracted index is contiguous, STEP bytes of a row at
// a time. Chunk c of a row sits at position c ^ swizzle(row) in LDS, so that the lanes
// that read one chunk of neighbouring rows reach different banks. PERM: fragment f of
// a block of 64 rows holds rows 16 (i / 4) + 4 f + i % 4 (i: the lane's row of 16) in
// place of 16 f + i, so that a lane's results of four fragments are 16 consecutive rows.
template <class T, int R, int NW, bool PERM, int STEP>
struct RowOperand {
  static constexpr int kChunks = STEP / 16;
  static constexpr int kLds = R * STEP;
  static constexpr int kLoads = R * kChunks / (NW * 64);
  static_assert(kLoads * NW * 64 == R * kChunks && (STEP == 64 || STEP == 128));
  __device__ static int swizzle(int row) {
    if constexpr (STEP == 128) return PERM ? (row & 3) | ((row >> 4) & 1) << 2 : row & 7;
    return PERM ? ((row >> 1) & 1) | ((row >> 4) & 1) << 1 : (row >> 1) & 3;
  }
  __device__ static int frag_row(int f, int i) {
    return PERM ? (f >> 2) * 64 + 16 * (i >> 2) + 4 * (f & 3) + (i & 3) : 16 * f + i;
  }

  const char* base;  // the tile's first row at the current step
  int64_t ld;        // bytes of a row
  int rows, left;    // rows in range; bytes of a row still in range
  uint32_t off[kLoads];  // of the thread's loads, from base on

  __device__ RowOperand(const void* p, int64_t ld_bytes, int rows_, int64_t length)
      : base(static_cast<const char*>(p)), ld(ld_bytes), rows(rows_), left((int)(length * T::kBytes)) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) off[i] = load_row(i) < rows ? row_offset(i) + load_at(i) : kOutOfRange;
    if (left < STEP) clip();
  }
  __device__ void advance(int steps = 1) {
    base = in_scalars(base + steps * STEP);
    left -= steps * STEP;
    if (left < STEP) clip();
  }
  __device__ void clip() {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) off[i] = load_at(i) < left ? off[i] : kOutOfRange;
  }
  // Load i of the thread: its row, and the chunk that goes to its position.
  __device__ static int load_row(int i) { return (i * NW * 64 + thread_of<NW>()) / kChunks; }
  __device__ static int load_at(int i) {
    return (((int)threadIdx.x & (kChunks - 1)) ^ swizzle(load_row(i))) * 16;
  }
  __device__ uint32_t row_offset(int i) const {  // past the last row any row will do
    const int row = load_row(i);
    return (uint32_t)(row < rows ? row : rows - 1) * (uint32_t)ld;
  }

  // Load i straight into LDS: rows of whole, aligned vectors; rows past the last, and
  // what is past a row's end, as zeros. First place, then fetch. ONCE: nobody else reads them.
  __device__ static void place(LdsPtr lds, int i) { lds_place(lds + (i * NW + wave_of<NW>()) * 1024); }
  template <bool ONCE = false>
  __device__ void fetch(int i) const {
    load_to_place<16, ONCE>(buffer_from(base), off[i]);
  }
  // Through registers: any alignment and length from 16 bytes.
  __device__ void load(u32x4 (&v)[kLoads]) const {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) v[i] = load_before_end(base + row_offset(i), load_at(i), left);
  }
  // What load brought `ago` steps ago, to LDS.
  __device__ void store(u32x4 (&v)[kLoads], LdsPtr lds, int ago) const {
    const int end = left + ago * STEP;
    if (end < STEP) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) v[i] = drop_bytes(v[i], over_end(load_at(i), end));
    }
#pragma unroll
    for (int i = 0; i < kLoads; ++i) lds_store(v[i], lds + (i * NW * 64 + thread_of<NW>()) * 16);
  }
  // Where in `lds` the lane's part of the fragments is whose rows begin at row0, and
  // fragment f of 64 bytes `ks` of the step: rows of other fragments swizzle alike.
  template <int F>
  struct Lane {
    int at[STEP / 64];
    __device__ Lane(LdsPtr lds, int row0) {
      const int lane = threadIdx.x & 63, row = row0 + frag_row(0, lane & 15);
#pragma unroll
      for (int ks = 0; ks < STEP / 64; ++ks) {
        at[ks] = in_vector((int)(uintptr_t)lds + row * STEP + ((ks * 4 + (lane >> 4)) ^ swizzle(row)) * 16);
      }
    }
    __device__ u32x4 fragment(int f, int ks, int further = 0) const {
      return lds_load<u32x4>((LdsPtr)(uintptr_t)(uint32_t)(at[ks] + further) + frag_row(f, 0) * STEP);
    }
  };
};

// An operand whose R rows are contiguous for one contracted index: a step is kDepth
// rows of memory, R elements of each. In LDS a chunk sits at position
// chunk ^ swizzle(c). 16-bit fragments are transposed by ds_read_b64_tr_b16 (lanes
// 4 j .. 4 j + 3 of 16 point at 16 elements of the j-th of four rows, and lane i
// receives the four rows' i-th elements); fp32 ones are read one by one.
template <class T, int R, int NW, int STEP>
struct ColOperand {
  static constexpr int kDepth = STEP / T::kBytes;
  static constexpr int kWide = R * T::kBytes / 16;  // chunks of a row in LDS
  static constexpr int kLds = R * STEP;
  static constexpr int kLoads = R * (STEP / 16) / (NW * 64);
  static_assert(kLoads * NW * 64 == R * (STEP / 16));
  // 32 bytes apart from row to row, and 128 from lane group to lane group (rows of 128
  // bytes: from row to row but one, and 64).
  __device__ static int swizzle(int c) {
    if constexpr (kWide == 8) return ((c >> 1) & 1) << 1 | ((c >> 3) & 1) << 2;
    return T::kBytes == 2 ? (c & 3) << 1 | ((c >> 3) & 1) << 3 : ((c >> 2) & 3) * 4;
  }
  static_assert(kWide >= 16 || (kWide == 8 && T::kBytes == 2));
  __device__ static int frag_row(int f, int i) { return 16 * f + i; }

  const char* base;  // the tile's first column at the current step
  int64_t ld;        // bytes of a row of memory
  int wide, left;    // bytes of it in the tile; contracted rows in range
  uint32_t off[kLoads];  // of the thread's loads, from base on

  __device__ ColOperand(const void* p, int64_t ld_bytes, int rows, int64_t length)
      : base(static_cast<const char*>(p)), ld(ld_bytes), wide(rows * T::kBytes), left((int)length) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      off[i] = load_at(i) < wide ? (uint32_t)load_c(i) * (uint32_t)ld + load_at(i) : kOutOfRange;
    }
    if (left < kDepth) clip();
  }
  __device__ void advance() {
    base = in_scalars(base + kDepth * ld);
    left -= kDepth;
    if (left < kDepth) clip();
  }
  __device__ void clip() {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) off[i] = load_c(i) < left ? off[i] : kOutOfRange;
  }
  __device__ static int load_c(int i) { return (i * NW * 64 + thread_of<NW>()) / kWide; }
  __device__ static int load_at(int i) { return (((int)threadIdx.x & (kWide - 1)) ^ swizzle(load_c(i))) * 16; }

  // Load i straight into LDS; rows past the last and chunks past the tile's columns as zeros.
  __device__ static void place(LdsPtr lds, int i) { lds_place(lds + (i * NW + wave_of<NW>()) * 1024); }
  template <bool ONCE = false>
  __device__ void fetch(int i) const {
    load_to_place<16, ONCE>(buffer_from(base), off[i]);
  }
  // A row past the last is the last; what a chunk holds past the tile's columns does
  // not matter, since nothing of it is stored.
  __device__ void load(u32x4 (&v)[kLoads]) const {
    const int last = left < kDepth ? left - 1 : kDepth - 1;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int c = load_c(i);
      v[i] = load_before_end(base + (int64_t)(c < last ? c : last) * ld, load_at(i), wide);
    }
  }
  __device__ void store(u32x4 (&v)[kLoads], LdsPtr lds, int ago) const {
    const int n = left + ago * kDepth;  // rows in range then
    if (wide < R * T::kBytes) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) v[i] = drop_bytes(v[i], over_end(load_at(i), wide));
    }
    if (n < kDepth) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) v[i] = load_c(i) < n ? v[i] : (u32x4){0u, 0u, 0u, 0u};
    }
#pragma unroll
    for (int i = 0; i < kLoads; ++i) lds_store(v[i], lds + (i * NW * 64 + thread_of<NW>()) * 16);
  }
  // As RowOperand's, of F fragments. They are 16 elements apart, and no other bit of row0
  // or the lane's column is as high, so that the swizzle's exclusive or takes them in.
  template <int F>
  struct Lane {
    int at[F];
    __device__ Lane(LdsPtr lds, int row0) {
      const int i = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4;
      const int c = T::kBytes == 2 ? g * 8 + (i >> 2) : g * 4, col = row0 + (T::kBytes == 2 ? 4 * (i & 3) : i);
      const int chunk = (col * T::kBytes / 16) ^ swizzle(c);
      const int first = (c * kWide + chunk) * 16 + col * T::kBytes % 16;
#pragma unroll
      for (int f = 0; f < F; ++f) at[f] = in_vector((int)(uintptr_t)lds + (first ^ (f * 16 * T::kBytes)));
    }
    __device__ u32x4 fragment(int f, int ks) const {
      constexpr int kRow = kWide * 16;
      const LdsPtr p = (LdsPtr)(uintptr_t)(uint32_t)at[f] + ks * (64 / T::kBytes) * kRow;
      if constexpr (T::kBytes == 2) {  // c + 4 swizzles as c
        using Lds4 = __attribute__((address_space(3))) s16x4*;
        const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<Lds4>(p)));
        const u32x2 b = __builtin_bit_cast(
            u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<Lds4>(p + 4 * kRow)));
        return (u32x4){a[0], a[1], b[0], b[1]};
      } else {
        u32x4 v;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = lds_load<uint32_t>(p + j * kRow);
        return v;
      }
    }
  };
};

// The E8M0 scales of an operand of R rows (`blocks` bytes a row): for each 64 bytes of
// a step four bytes a row, one for each chunk. A wave's rows are in the order of its
// lanes and then its F fragments, so that a lane reads its fragments' as vectors.
template <class Operand, int R, int NW, int F, int STEP>
struct Scales {
  static constexpr int kHalves = STEP / 64, kWords = R * kHalves;
  static constexpr int kLoads = (kWords + NW * 64 - 1) / (NW * 64);
  static constexpr int kLds = kLoads * NW * 256;
  const char* base;
  int64_t ld;
  int rows, left;

  __device__ Scales(const void* p, int64_t blocks, int rows_)
      : base(static_cast<const char*>(p)), ld(blocks), rows(rows_), left((int)blocks) {}
  __device__ void advance(int steps = 1) {
    base += steps * STEP / 16;
    left -= steps * STEP / 16;
  }
  // Word i of the thread: [half][wave's rows][lane][fragment].
  __device__ static int load_at(int i) { return (i * NW * 64 + thread_of<NW>()) / R * 4; }
  __device__ uint32_t row_offset(int i) const {
    const int d = (i * NW * 64 + thread_of<NW>()) % R, in = d % (F * 16);
    const int row = d - in + Operand::frag_row(in % F, in / F);
    return (uint32_t)(row < rows ? row : rows - 1) * (uint32_t)ld;
  }
  __device__ static void place(LdsPtr lds, int i) { lds_place(lds + (i * NW + wave_of<NW>()) * 256); }
  __device__ void fetch(int i) const {
    const int at = load_at(i);
    load_to_place<4, false>(buffer_from(base), at < left ? row_offset(i) + at : kOutOfRange);
  }
  // Any alignment and number of blocks. Past the last block its scale is as good as
  // any: the codes there are zeros, and a row whose last scale is NaN is NaN.
  __device__ void load(uint32_t (&v)[kLoads]) const {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const char* p = base + row_offset(i);
      v[i] = 0u;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = load_at(i) + j;
        v[i] |= (uint32_t)(uint8_t)p[k < left ? k : left - 1] << (8 * j);
      }
    }
  }
  __device__ static void store(const uint32_t (&v)[kLoads], LdsPtr lds) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) lds_store(v[i], lds + (i * NW * 64 + thread_of<NW>()) * 4);
  }
  // The scales of the lane's rows of all fragments, four of a row each; of_lane takes
  // the lane's to the low byte.
  __device__ static void read(LdsPtr lds, int row0, int (&s)[F], int half) {
    const int lane = threadIdx.x & 63;
    const LdsPtr p = lds + (half * R + row0 + (lane & 15) * F) * 4;
    if constexpr (F % 4 == 0) {
#pragma unroll
      for (int f = 0; f < F; f += 4) {
        const u32x4 v = lds_load<u32x4>(p + f * 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) s[f + j] = (int)v[j];
      }
    } else {
#pragma unroll
      for (int f = 0; f < F; ++f) s[f] = lds_load<int>(p + f * 4);
    }
  }
  __device__ static void of_lane(const int (&s)[F], int (&mine)[F]) {
#pragma unroll
    for (int f = 0; f < F; ++f) mine[f] = (int)((uint32_t)s[f] >> (8 * ((threadIdx.x & 63) >> 4)));
  }
};

// In place of the scales of the types that have none.
struct NoScales {
  static constexpr int kLds = 0, kLoads = 0;
  __device__ void advance(int = 1) {}
  __device__ static void place(LdsPtr, int) {}
  __device__ void fetch(int) const {}
  __device__ void load(uint32_t (&)[1]) const {}
  __device__ static void store(const uint32_t (&)[1], LdsPtr) {}
  template <int F>
  __device__ static void read(LdsPtr, int, int (&)[F], int) {}
  template <int F>
  __device__ static void of_lane(const int (&)[F], int (&)[F]) {}
};

// ---------------------------------------------------------------------------
// The product.
// ---------------------------------------------------------------------------

// Sums of fragments, and their folding for the types that need it.
template <class T, int FP, int FQ>
struct Folded {
  f32x4 sum[T::kFold ? FP : 1][T::kFold ? FQ : 1] = {};
  __device__ void fold(f32x4 (&acc)[FP][FQ]) {
    if constexpr (T::kFold != 0) {
#pragma unroll
      for (int i = 0; i < FP; ++i) {
#pragma unroll
        for (int j = 0; j < FQ; ++j) {
          sum[i][j] += acc[i][j];
          acc[i][j] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
        }
      }
    }
  }
  // After so many halves of steps, two or four at a time.
  __device__ void every(int halves, f32x4 (&acc)[FP][FQ]) {
    if constexpr (T::kFold != 0) {
      if (halves % T::kFold == 0) fold(acc);
    }
  }
  __device__ void end(f32x4 (&acc)[FP][FQ]) const {
    if constexpr (T::kFold != 0) {
#pragma unroll
      for (int i = 0; i < FP; ++i) {
#pragma unroll
        for (int j = 0; j < FQ; ++j) acc[i][j] += sum[i][j];
      }
    }
  }
};

// ONCE: Q's loads as of data that no other workgroup reads.
template <class T, class P, class Q, class PS, class QS, int WP, int WQ, int FP, int FQ, int STEP, bool ONCE = false>
struct Product {
  static constexpr bool kDirect = STEP == 128;  // straight into LDS, or (64) through registers
  static constexpr int kSlots = kDirect ? 2 : 4;
  // Of a slot: P, Q, the scales of P and of Q.
  static constexpr int kAtQ = P::kLds, kAtPS = kAtQ + Q::kLds, kAtQS = kAtPS + PS::kLds, kSlot = kAtQS + QS::kLds;
  static constexpr int kLds = kSlots * kSlot;

  // Where a wave's fragments are in a slot: rows from p0, columns from q0 on.
  struct Lanes {
    LdsPtr slot;
    int p0, q0;
    typename P::template Lane<FP> p;
    typename Q::template Lane<FQ> q;
    __device__ Lanes(LdsPtr slot_, int p0_, int q0_)
        : slot(slot_), p0(p0_), q0(q0_), p(slot_, p0_), q(slot_ + kAtQ, q0_) {}
  };

  // acc[fp][fq] += the product over `steps` > 0 steps of the wave's rows from p0 and
  // columns from q0 on; lds: kLds bytes, which are free again behind it. All waves of the
  // workgroup call, or idle.
  __device__ static void run(const P& p, const Q& q, const PS& ps, const QS& qs, int steps, LdsPtr lds, int p0, int q0,
                             f32x4 (&acc)[FP][FQ]) {
    if constexpr (kDirect) {
      direct(p, q, ps, qs, steps, lds, p0, q0, acc);
    } else {
      through_registers(p, q, ps, qs, steps, lds, p0, q0, acc);
    }
  }

  // For a wave whose part of the tile is past its rows or columns: it loads its share,
  // and leaves the matrix cores to the others, so that a tile that is at most half
  // filled takes about half the time.
  __device__ static void idle(P p, Q q, PS ps, QS qs, int steps, LdsPtr lds) {
    if constexpr (kDirect) {
      Asking ask{p, q, ps, qs};
      ask.all(lds);
      ask.all(lds + kSlot);
      loads_landed<Asking::kAll>();
      meet();
      for (int t = 0; t < looped(steps); ++t) {
        meet();
        ask.all(lds + (t & 1) * kSlot);
        loads_landed<Asking::kAll>();
        meet();
      }
      loads_landed();
      meet();
    } else {
      f32x4 acc[FP][FQ] = {};
      through_registers(p, q, ps, qs, steps, lds, 0, 0, acc);
    }
  }

  // Half a step's products are issued in kParts parts, with reads and loads between them:
  // one by one where a SIMD has a single wave to issue anything (kWide), else by rows.
  // 256 x 256 tiles of rows take 2215 cycles a step so, of which the matrix cores need 2048; with
  // Q in columns 2280, with both 2360; and 27000 beside the steps, the launch among them (slopes
  // of 56 to 224 steps, one tile a CU). 8192 rows on 8 groups of 14336 x 4096, bf16: 790 us,
  // 1.22 PFLOP/s; 128 x 128 tiles, two workgroups a CU, which LDS bounds, 1057.
  static constexpr bool kWide = FP == 8 && FQ == 8;
  // Sums in the accumulation registers: for the wide ones, and for the scaled products, whose
  // builtin takes operands of twice the size, zeros behind what there is of them.
  static constexpr bool kSumsApart = kWide || (kDirect && T::kScaled);
  static constexpr int kParts = kWide ? FP * FQ : FP;
  // In half 1 the reads take the first parts, and the loads all behind the barrier, of both halves.
  static constexpr int kReadParts = kWide ? 20 : (kParts + 3) / 4;
  static constexpr int kMeetPart = kParts == 2 ? 1 : kReadParts + (kParts + 15) / 16;
  static_assert(kReadParts <= kMeetPart && kMeetPart < kParts);
  static constexpr int kAskParts = 2 * kParts - kMeetPart;
  // fn(i) for the items i of `items` that part `part` of `parts` takes, spread evenly.
  template <class Fn>
  __device__ static void spread(int items, int part, int parts, Fn&& fn) {
#pragma unroll
    for (int i = part * items / parts; i < (part + 1) * items / parts; ++i) fn(i);
  }

  // What 64 bytes a row multiply.
  struct Fragments {
    u32x4 p[FP], q[FQ];
    int sp[FP], sq[FQ];
    __device__ void read(const Lanes& at, int ks, int part, int parts) {
      if (part == 0) {
        QS::read(at.slot + kAtQS, at.q0, sq, ks);
        PS::read(at.slot + kAtPS, at.p0, sp, ks);
      }
      spread(FP + FQ, part, parts, [&](int i) {
        if (i < FQ) {
          q[i] = at.q.fragment(i, ks);
        } else {
          p[i - FQ] = at.p.fragment(i - FQ, ks);
        }
      });
    }
    __device__ void read(const Lanes& at, int ks) { read(at, ks, 0, 1); }
    // between(part) is issued before the part's products.
    template <class Fn>
    __device__ void multiply(f32x4 (&acc)[FP][FQ], Fn&& between) const {
      __builtin_amdgcn_sched_barrier(0);
      int mp[FP] = {}, mq[FQ] = {};
      PS::of_lane(sp, mp);
      QS::of_lane(sq, mq);
      if constexpr (kSumsApart) {
        if constexpr (T::kScaled) computed_here(mp), computed_here(mq);
        operands_ready();
      }
#pragma unroll
      for (int part = 0; part < kParts; ++part) {
        between(part);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (kWide) {
          const int a = part / FQ, b = part % FQ;
          T::mma_acc(q[b], p[a], acc[a][b], mq[b], mp[a]);
        } else {
#pragma unroll
          for (int b = 0; b < FQ; ++b) {
            if constexpr (kSumsApart) {
              T::mma_acc(q[b], p[part], acc[part][b], mq[b], mp[part]);
            } else {
              acc[part][b] = T::mma(q[b], p[part], acc[part][b], mq[b], mp[part]);
            }
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };

  // The loads of a step; those of a step past the last bring zeros.
  struct Asking {
    P p;
    Q q;
    PS ps;
    QS qs;
    static constexpr int kP = P::kLoads, kQ = kP + Q::kLoads, kPS = kQ + PS::kLoads, kAll = kPS + QS::kLoads;
    // Load i: its place, and the load itself.
    __device__ void place(LdsPtr to, int i) const {
      if (i < kP) {
        P::place(to, i);
      } else if (i < kQ) {
        Q::place(to + kAtQ, i - kP);
      } else if (i < kPS) {
        PS::place(to + kAtPS, i - kQ);
      } else {
        QS::place(to + kAtQS, i - kPS);
      }
    }
    __device__ void fetch(int i) const {
      if (i < kP) {
        p.fetch(i);
      } else if (i < kQ) {
        q.template fetch<ONCE>(i - kP);
      } else if (i < kPS) {
        ps.fetch(i - kQ);
      } else {
        qs.fetch(i - kPS);
      }
    }
    // Part `part` of kAskParts of them. Where there are parts enough, a load's two
    // instructions are in two of them, with products between.
    __device__ void part(LdsPtr to, int part) const {
      if constexpr (kWide) {
        spread(2 * kAll, part, kAskParts, [&](int i) {
          if (i % 2 == 0) {
            place(to, i / 2);
          } else {
            fetch(i / 2);
          }
        });
      } else {
        spread(kAll, part, kAskParts, [&](int i) { one(to, i); });
      }
    }
    __device__ void one(LdsPtr to, int i) const {
      place(to, i);
      place_ready();
      fetch(i);
    }
    // Loads whose instructions are all in the first `parts` parts.
    static constexpr int issued(int parts) {
      return kWide ? 2 * kAll * parts / kAskParts / 2 : kAll * parts / kAskParts;
    }
    __device__ void advance() {
      p.advance();
      q.advance();
      ps.advance();
      qs.advance();
    }
    __device__ void all(LdsPtr to) {
#pragma unroll
      for (int i = 0; i < kAll; ++i) one(to, i);
      advance();
    }
  };

  // The wide loop has no other exit: an odd last step is followed by one of zeros.
  __device__ static int looped(int steps) { return kWide ? (steps + 1) / 2 * 2 : steps / 2 * 2; }

  __device__ static void direct(const P& p, const Q& q, const PS& ps, const QS& qs, int steps, LdsPtr lds, int p0,
                                int q0, f32x4 (&acc)[FP][FQ]) {
    Asking ask{p, q, ps, qs};
    Fragments first, second;
    Folded<T, FP, FQ> folded;
    const LdsPtr lds1 = lds + kSlot;
    const Lanes at0(lds, p0, q0), at1(lds1, p0, q0);
    auto step = [&](const Lanes& now, const Lanes& next) {
      first.multiply(acc, [&](int part) {
        if (part < kReadParts) second.read(now, 1, part, kReadParts);
        if (part == kMeetPart) {
          lds_read();
          meet();
        }
        if (part >= kMeetPart) ask.part(now.slot, part - kMeetPart);
      });
      loads_landed<Asking::issued(kParts - kMeetPart)>();
      meet();
      second.multiply(acc, [&](int part) {
        first.read(next, 0, part, kParts);
        ask.part(now.slot, kParts - kMeetPart + part);
      });
      ask.advance();
    };
    ask.all(lds);
    ask.all(lds1);
    loads_landed<Asking::kAll>();
    meet();
    first.read(at0, 0);
    const int whole = looped(steps);
    int t = 0;
    auto two = [&] {
      step(at0, at1);
      step(at1, at0);
      t += 2;
      folded.every(2 * t, acc);
    };
    if constexpr (kWide) {
      // At least once, as steps > 0: with a way around the loop the compiler copies the sums where
      // both ways meet, in front of the wait that acc_ready is.
      do {
        two();
      } while (t < whole);
    } else {
      while (t < whole) two();
      if (t < steps) {
        second.read(at0, 1);
        first.multiply(acc, [](int) {});
        second.multiply(acc, [](int) {});
      }
    }
    loads_landed();
    meet();  // nobody reads the slots any more, and nothing is on its way to them
    if constexpr (kSumsApart) acc_ready(acc);
    folded.end(acc);
  }

  // With loads that wait in registers, two steps of them; a ring of four slots.
  __device__ static void through_registers(P p, Q q, PS ps, QS qs, int steps, LdsPtr lds, int p0, int q0,
                                           f32x4 (&acc)[FP][FQ]) {
    Fragments frag;
    Folded<T, FP, FQ> folded;
    struct Held {
      u32x4 p[P::kLoads], q[Q::kLoads];
      uint32_t ps[PS::kLoads ? PS::kLoads : 1], qs[QS::kLoads ? QS::kLoads : 1];
    } even, odd;
    auto load = [&](Held& h) {
      p.load(h.p);
      q.load(h.q);
      ps.load(h.ps);
      qs.load(h.qs);
      p.advance();
      q.advance();
      ps.advance();
      qs.advance();
    };
    auto store = [&](Held& h, int slot, int ago) {
      const LdsPtr s = lds + slot * kSlot;
      p.store(h.p, s, ago);
      q.store(h.q, s + kAtQ, ago);
      PS::store(h.ps, s + kAtPS);
      QS::store(h.qs, s + kAtQS);
    };
    auto step = [&](Held& h, int slot) {
      store(h, slot, 2);
      __syncthreads();
      load(h);
      frag.read(Lanes(lds + slot * kSlot, p0, q0), 0);
      frag.multiply(acc, [](int) {});
    };
    load(even);
    load(odd);
    int t = 0;
    for (; t + 2 <= steps; t += 2) {
      step(even, t & 2);
      step(odd, (t & 2) + 1);
      folded.every(t + 2, acc);
    }
    if (t < steps) step(even, t & 2);
    __syncthreads();  // nobody reads the slots any more
    folded.end(acc);
  }
};

template <class S>
__device__ inline S scales_of(const char* p, int64_t blocks, int rows) {
  if constexpr (std::is_same_v<S, NoScales>) {
    return S();
  } else {
    return S(p, blocks, rows);
  }
}

// Zeros in the workgroup's tile of NW waves: `rows` rows of `cols` columns.
template <class C, int NW>
__device__ inline void store_zeros(char* out, int64_t ld, int rows, int cols) {
  const u32x4 zeros = {0u, 0u, 0u, 0u};
  const int chunks = (cols + C::VEC - 1) / C::VEC;
  for (int i = threadIdx.x; i < rows * chunks; i += NW * 64) {
    const int row = i / chunks, q = (i - row * chunks) * C::VEC;
    char* const to = out + ((int64_t)row * ld + q) * C::kBytes;
    if (q + C::VEC <= cols) {
      __builtin_nontemporal_store(zeros, reinterpret_cast<u32x4_any*>(to));
    } else {
      store_partial<C>(zeros, cols - q, to);
    }
  }
}

// Stores a wave's fragments: rows [p0, rows) of `out` (row stride ld elements), columns
// [q0, cols). Straight from the registers a store would take 16 or 8 bytes of each of 16
// rows. So the wave turns its part over in `lds`, SPACE bytes that it keeps to itself, and
// stores take whole rows of it (weight gradient of 8192 rows, 8 experts of 14336 x 4096: 937
// us, 1006 straight), past the caches (64 experts of 96 rows, 1408 x 2048: 108 us, 144
// through them). Vectors are stored at any byte.
template <class C, bool PERM, int FP, int FQ, int SPACE>
__device__ inline void store_tile(const f32x4 (&acc)[FP][FQ], LdsPtr lds, char* out, int64_t ld, int p0, int q0,
                                  int rows, int cols) {
  constexpr int kRow = FQ * 16 * C::kBytes, kChunks = kRow / 16;  // of a row of the part
  constexpr int kFrags = SPACE / (16 * kRow) < FP ? SPACE / (16 * kRow) : FP;  // turned over at a time
  static_assert(kFrags >= 1 && FP % kFrags == 0 && 64 % kChunks == 0);
  constexpr int kRun = PERM ? 16 : 4;  // consecutive columns of a lane
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
#pragma unroll
  for (int a0 = 0; a0 < FP; a0 += kFrags) {
    if (p0 + 16 * a0 >= rows) break;
#pragma unroll
    for (int a = 0; a < kFrags; ++a) {
      const int row = 16 * a + i;
#pragma unroll
      for (int b = 0; b < FQ; b += kRun / 4) {
        const int at = (PERM ? (b >> 2) * 64 + 16 * g : 16 * b + 4 * g) * C::kBytes;  // bytes into the row
        float f[kRun < C::VEC ? C::VEC : kRun] = {};
#pragma unroll
        for (int j = 0; j < kRun; ++j) f[j] = acc[a0 + a][b + j / 4][j % 4];
#pragma unroll
        for (int v = 0; v < (kRun + C::VEC - 1) / C::VEC; ++v) {
          float part[C::VEC];
#pragma unroll
          for (int j = 0; j < C::VEC; ++j) part[j] = f[v * C::VEC + j];
          const u32x4 w = C::pack(part);
          const LdsPtr to = lds + row * kRow + ((((at >> 4) + v) ^ (row & (kChunks - 1))) << 4);
          if constexpr (kRun * C::kBytes >= 16) {
            lds_store(w, to);
          } else {
            lds_store((u32x2){w[0], w[1]}, to + (at & 8));
          }
        }
      }
    }
#pragma unroll 8
    for (int r = 0; r < kFrags * 16; r += 64 / kChunks) {
      const int row = r + lane / kChunks, chunk = lane % kChunks;
      const u32x4 w = lds_load<u32x4>(lds + row * kRow + ((chunk ^ (row & (kChunks - 1))) << 4));
      const int p = p0 + 16 * a0 + row, q = q0 + chunk * C::VEC;
      char* const to = out + ((int64_t)p * ld + q) * C::kBytes;
      if (p < rows) {
        if (q + C::VEC <= cols) {
          __builtin_nontemporal_store(w, reinterpret_cast<u32x4_any*>(to));
        } else if (q < cols) {
          store_partial<C>(w, cols - q, to);
        }
      }
    }
  }
}

// A few fragments, straight from the registers.
template <class C>
__device__ inline void store_fragment(const f32x4& acc, char* out, int64_t ld, int p0, int q0, int rows, int cols) {
  const int lane = threadIdx.x & 63, p = p0 + (lane & 15), q = q0 + 4 * (lane >> 4);
  if (p >= rows || q >= cols) return;
  float f[C::VEC] = {};
#pragma unroll
  for (int j = 0; j < 4; ++j) f[j] = acc[j];
  const u32x4 w = C::pack(f);
  char* const to = out + ((int64_t)p * ld + q) * C::kBytes;
  if (q + 4 > cols) {
    store_partial<C>(w, cols - q, to);
  } else if constexpr (C::kBytes == 4) {
    *reinterpret_cast<u32x4_any*>(to) = w;
  } else {
    *reinterpret_cast<u32x2_any*>(to) = (u32x2){w[0], w[1]};
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
  int first;  // the tile of the launch's first workgroup
};

// Waves on a SIMD that a tile of so many fragments a wave leaves registers for: two
// (256 a lane) for 16. 64, and tiles that go through registers, need more.
constexpr int tile_waves(int fragments, bool direct) { return direct && fragments <= 16 ? 2 : 1; }

template <class T, class C, bool QROWS, int WP, int WQ, int FP, int FQ, bool DIRECT, bool ONCE>
__global__ __launch_bounds__(WP* WQ * 64, tile_waves(FP* FQ, DIRECT)) void rows_product(RowsArgs a) {
  constexpr int BP = WP * FP * 16, BQ = WQ * FQ * 16, NW = WP * WQ, kStep = DIRECT ? 128 : 64;
  using P = RowOperand<T, BP, NW, false, kStep>;
  constexpr bool kPerm = QROWS && FQ % 4 == 0;
  using Q = std::conditional_t<QROWS, RowOperand<T, BQ, NW, kPerm, kStep>, ColOperand<T, BQ, NW, kStep>>;
  using PS = std::conditional_t<T::kScaled, Scales<P, BP, NW, FP, kStep>, NoScales>;
  using QS = std::conditional_t<T::kScaled, Scales<Q, BQ, NW, FQ, kStep>, NoScales>;
  using Prod = Product<T, P, Q, PS, QS, WP, WQ, FP, FQ, kStep, ONCE>;
  __shared__ __attribute__((aligned(1024))) char lds[Prod::kLds];
  __shared__ typename RowTiles<BP, NW * 64>::Shared shared;

  // Row tiles that mostly are of groups apart share no weights: one group's are read in one run.
  constexpr int kHeight = ONCE ? 2 : 8;
  RowTileAt at;
  int tp, tq;
  const int id = a.first + (int)blockIdx.x;
  if (a.offsets != nullptr) {
    const RowTiles<BP, NW * 64> tiles(shared, a.offsets, a.groups, a.rows, a.most);
    const int total = tiles.total * a.tiles_q;
    if (id >= total) return;
    tile_order<kHeight>(xcd_contiguous(id, total), tiles.total, a.tiles_q, &tp, &tq);
    at = tiles.at(tp);
    if (at.count == 0) return;
  } else {
    tile_order<kHeight>(xcd_contiguous(id, a.most * a.tiles_q), a.most, a.tiles_q, &tp, &tq);
    at.row = (int64_t)tp * BP;
    at.count = a.rows - at.row < BP ? (int)(a.rows - at.row) : BP;
    at.group = 0;
  }

  const int col = tq * BQ, width = a.cols - col < BQ ? a.cols - col : BQ;
  const int wave = wave_of<NW>(), p0 = (wave / WQ) * FP * 16, q0 = (wave % WQ) * FQ * 16;
  char* const out = a.out + (at.row * a.cols + col) * C::kBytes;
  if (at.group < 0) {
    store_zeros<C, NW>(out, a.cols, at.count, width);
    return;
  }
  const int64_t e = at.group, ldp = a.length * T::kBytes, ldq = QROWS ? ldp : (int64_t)a.cols * T::kBytes;
  const char* wt = a.w + e * a.length * a.cols * T::kBytes + (QROWS ? col * ldq : (int64_t)col * T::kBytes);
  const int steps = (int)((ldp + kStep - 1) / kStep);
  const P p(a.x + at.row * ldp, ldp, at.count, a.length);
  const Q q(wt, ldq, width, a.length);
  const int64_t blocks = a.length / 16;
  const PS ps = scales_of<PS>(a.x_scale + at.row * blocks, blocks, at.count);
  const QS qs = scales_of<QS>(a.w_scale + (e * a.cols + col) * blocks, blocks, width);
  if (p0 >= at.count || q0 >= width) {
    Prod::idle(p, q, ps, qs, steps, (LdsPtr)lds);
    return;
  }
  f32x4 acc[FP][FQ] = {};
  Prod::run(p, q, ps, qs, steps, (LdsPtr)lds, p0, q0, acc);
  store_tile<C, kPerm, FP, FQ, Prod::kLds / NW>(acc, (LdsPtr)lds + wave * (Prod::kLds / NW), out, a.cols, p0, q0,
                                                at.count, width);
}

// ---------------------------------------------------------------------------
// Few rows a group: the weights are read once, and that is the time. A workgroup
// owns FP x 16 rows and FQ x 16 columns; its NW waves take the contracted index in
// turn, and their sums meet in LDS at the end, in the order of the waves. 16 rows on 8
// groups of 14336 x 4096, bf16: 113 us (their reads from HBM alone, at 6.9 TB/s, 123); straight
// from memory to registers, as rows off their alignment take, 160 to 200. A ring of two steps was
// as good as any deeper one, and 32 columns a workgroup of four waves as good as other shapes.
// ---------------------------------------------------------------------------

constexpr int kStreamBytes = 256, kStreamSteps = kStreamBytes / 64;

// A lane's chunks of a block of 16 x F rows, which may begin at any byte and have 16 or more.
template <class T, int F>
struct StreamOperand {
  const char* row[F];    // the lane's row of each fragment
  const char* scale[F];  // and its scales
  int bytes;             // of a row

  __device__ StreamOperand(const char* base, const char* scales, int64_t ld, int rows) : bytes((int)ld) {
    const int i = threadIdx.x & 15;
#pragma unroll
    for (int f = 0; f < F; ++f) {
      const int r = 16 * f + i < rows ? 16 * f + i : rows - 1;  // past the last row any row will do
      row[f] = base + (int64_t)r * ld;
      scale[f] = T::kScaled ? scales + (int64_t)r * (ld / 16) : nullptr;
    }
  }
  // LAST: the row's end cuts the block; zeros past it.
  template <bool LAST>
  __device__ void load(int block, u32x4 (&v)[F][kStreamSteps], int (&s)[F][kStreamSteps]) const {
    const int at = block * kStreamBytes + ((threadIdx.x >> 4) & 3) * 16;
#pragma unroll
    for (int f = 0; f < F; ++f) {
#pragma unroll
      for (int u = 0; u < kStreamSteps; ++u) {
        const int c = at + u * 64;
        if constexpr (LAST) {
          v[f][u] = drop_bytes(load_before_end(row[f], c, bytes), over_end(c, bytes));
        } else {
          v[f][u] = *reinterpret_cast<const u32x4_any*>(row[f] + c);
        }
        // Past the last block its scale is as good as any (see Scales::load).
        if constexpr (T::kScaled) s[f][u] = (uint8_t)scale[f][(c < bytes ? c : bytes - 16) >> 4];
      }
    }
  }
};

// acc += this wave's blocks, straight from memory to registers: a lane's chunk is a
// fragment as it is.
template <class T, int FP, int FQ, int NW>
__device__ inline void stream_direct(const char* x, const char* xs, int rows, const char* w, const char* ws, int cols,
                                     int64_t ld, int wave, f32x4 (&acc)[FP][FQ]) {
  const StreamOperand<T, FP> p(x, xs, ld, rows);
  const StreamOperand<T, FQ> q(w, ws, ld, cols);
  u32x4 pa[FP][kStreamSteps], qa[FQ][kStreamSteps], pb[FP][kStreamSteps], qb[FQ][kStreamSteps];
  int psa[FP][kStreamSteps], qsa[FQ][kStreamSteps], psb[FP][kStreamSteps], qsb[FQ][kStreamSteps];
  Folded<T, FP, FQ> folded;
  auto multiply = [&](const u32x4(&pv)[FP][kStreamSteps], const u32x4(&qv)[FQ][kStreamSteps],
                      const int(&ps)[FP][kStreamSteps], const int(&qs)[FQ][kStreamSteps]) {
#pragma unroll
    for (int u = 0; u < kStreamSteps; ++u) {
#pragma unroll
      for (int i = 0; i < FP; ++i) {
#pragma unroll
        for (int j = 0; j < FQ; ++j) {
          acc[i][j] = T::mma(qv[j][u], pv[i][u], acc[i][j], T::kScaled ? qs[j][u] : 0, T::kScaled ? ps[i][u] : 0);
        }
      }
    }
    folded.fold(acc);
  };
  // Blocks wave, wave + NW, ...: one on its way (the last once more, if need be) while one is multiplied.
  const int whole = (int)(ld / kStreamBytes);
  int b = wave;
  if (b < whole) {
    p.template load<false>(b, pa, psa);
    q.template load<false>(b, qa, qsa);
    for (; b + NW < whole; b += 2 * NW) {
      const int third = b + 2 * NW < whole ? b + 2 * NW : b;
      p.template load<false>(b + NW, pb, psb);
      q.template load<false>(b + NW, qb, qsb);
      __builtin_amdgcn_sched_barrier(0);  // loads first
      multiply(pa, qa, psa, qsa);
      p.template load<false>(third, pa, psa);
      q.template load<false>(third, qa, qsa);
      __builtin_amdgcn_sched_barrier(0);
      multiply(pb, qb, psb, qsb);
    }
    if (b < whole) multiply(pa, qa, psa, qsa);
  }
  if (whole * kStreamBytes < ld && wave == whole % NW) {
    p.template load<true>(whole, pa, psa);
    q.template load<true>(whole, qa, qsa);
    multiply(pa, qa, psa, qsa);
  }
  folded.end(acc);
}

// acc += this wave's steps of 128 bytes a row, through a ring of DEPTH steps in LDS
// that the wave keeps to itself: loads take whole 128-byte lines of eight rows.
template <class T, int FP, int FQ, int NW, int DEPTH>
struct StreamRing {
  static constexpr int kStep = 128;
  using P = RowOperand<T, FP * 16, 1, false, kStep>;
  using Q = RowOperand<T, FQ * 16, 1, false, kStep>;
  using PS = std::conditional_t<T::kScaled, Scales<P, FP * 16, 1, FP, kStep>, NoScales>;
  using QS = std::conditional_t<T::kScaled, Scales<Q, FQ * 16, 1, FQ, kStep>, NoScales>;
  static constexpr int kAtQ = P::kLds, kAtPS = kAtQ + Q::kLds, kAtQS = kAtPS + PS::kLds, kSlot = kAtQS + QS::kLds;
  static constexpr int kLds = DEPTH * kSlot;
  static constexpr int kLoads = P::kLoads + Q::kLoads + PS::kLoads + QS::kLoads;  // of a step

  __device__ static void run(const char* x, const char* xs, int rows, const char* w, const char* ws, int cols,
                             int64_t length, int wave, LdsPtr lds, f32x4 (&acc)[FP][FQ]) {
    const int64_t ld = length * T::kBytes;
    P p(x, ld, rows, length);
    Q q(w, ld, cols, length);
    PS ps = scales_of<PS>(xs, ld / 16, rows);
    QS qs = scales_of<QS>(ws, ld / 16, cols);
    const int total = (int)((ld + kStep - 1) / kStep), steps = (total - wave + NW - 1) / NW;
    auto advance = [&](int n) {
      p.advance(n);
      q.advance(n);
      ps.advance(n);
      qs.advance(n);
    };
    auto ask = [&](LdsPtr to) {  // a step past the end is zeros
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
#pragma unroll
      for (int i = 0; i < PS::kLoads; ++i) {
        PS::place(to + kAtPS, i);
        place_ready();
        ps.fetch(i);
      }
#pragma unroll
      for (int i = 0; i < QS::kLoads; ++i) {
        QS::place(to + kAtQS, i);
        place_ready();
        qs.fetch(i);
      }
      advance(NW);
    };
    advance(wave);
    const typename P::template Lane<FP> p_lane(lds, 0);
    const typename Q::template Lane<FQ> q_lane(lds + kAtQ, 0);
    Folded<T, FP, FQ> folded;
    for (int d = 0; d < DEPTH; ++d) ask(lds + d * kSlot);
    int slot = 0;
    for (int t = 0; t < steps; ++t) {
      const LdsPtr from = lds + slot * kSlot;
      u32x4 pf[2][FP], qf[2][FQ];
      int rp[2][FP], rq[2][FQ];
      loads_landed<(DEPTH - 1) * kLoads>();
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
        for (int f = 0; f < FQ; ++f) qf[ks][f] = q_lane.fragment(f, ks, slot * kSlot);
#pragma unroll
        for (int f = 0; f < FP; ++f) pf[ks][f] = p_lane.fragment(f, ks, slot * kSlot);
        QS::read(from + kAtQS, 0, rq[ks], ks);
        PS::read(from + kAtPS, 0, rp[ks], ks);
      }
      lds_read();
      ask(from);
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        int sp[FP] = {}, sq[FQ] = {};
        PS::of_lane(rp[ks], sp);
        QS::of_lane(rq[ks], sq);
#pragma unroll
        for (int i = 0; i < FP; ++i) {
#pragma unroll
          for (int j = 0; j < FQ; ++j) acc[i][j] = T::mma(qf[ks][j], pf[ks][i], acc[i][j], sq[j], sp[i]);
        }
      }
      slot = slot + 1 < DEPTH ? slot + 1 : 0;
      folded.every(2 * (t + 1), acc);
    }
    loads_landed();
    folded.end(acc);
  }
};

template <class T, class C, int FP, int FQ, int NW, int DEPTH>
__global__ __launch_bounds__(NW * 64, DEPTH ? 1 : 2) void rows_stream(RowsArgs a) {
  constexpr int BP = FP * 16, BQ = FQ * 16;
  using Ring = StreamRing<T, FP, FQ, NW, DEPTH>;
  constexpr int kSums = NW * FP * FQ * 1024;
  __shared__ __attribute__((aligned(1024))) char lds[NW * Ring::kLds > kSums ? NW * Ring::kLds : kSums];
  __shared__ typename RowTiles<BP, NW * 64>::Shared shared;

  RowTileAt at;
  int tp, tq;
  const int id = a.first + (int)blockIdx.x;
  if (a.offsets != nullptr) {
    const RowTiles<BP, NW * 64> tiles(shared, a.offsets, a.groups, a.rows, a.most);
    const int total = tiles.total * a.tiles_q;
    if (id >= total) return;
    tile_order(xcd_contiguous(id, total), tiles.total, a.tiles_q, &tp, &tq);
    at = tiles.at(tp);
    if (at.count == 0) return;
  } else {
    tile_order(xcd_contiguous(id, a.most * a.tiles_q), a.most, a.tiles_q, &tp, &tq);
    at.row = (int64_t)tp * BP;
    at.count = a.rows - at.row < BP ? (int)(a.rows - at.row) : BP;
    at.group = 0;
  }

  const int col = tq * BQ, width = a.cols - col < BQ ? a.cols - col : BQ;
  const int64_t e = at.group < 0 ? 0 : at.group, ld = a.length * T::kBytes, blocks = ld / 16;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  f32x4 acc[FP][FQ] = {};
  if (at.group >= 0) {
    const char *xs = a.x_scale + at.row * blocks, *ws = a.w_scale + (e * a.cols + col) * blocks;
    if constexpr (DEPTH > 0) {
      Ring::run(a.x + at.row * ld, xs, at.count, a.w + (e * a.cols + col) * ld, ws, width, a.length, wave,
                (LdsPtr)lds + wave * Ring::kLds, acc);
    } else {
      stream_direct<T, FP, FQ, NW>(a.x + at.row * ld, xs, at.count, a.w + (e * a.cols + col) * ld, ws, width, ld, wave,
                                   acc);
    }
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
    store_fragment<C>(sum, a.out + (at.row * a.cols + col) * C::kBytes, a.cols, 16 * (f / FQ), 16 * (f % FQ), at.count,
                      width);
  }
}

// ---------------------------------------------------------------------------
// Rows of fewer than 16 bytes, in any operand: a wave an element of the output, its
// lanes over the contracted index. D[p][q] = sum_c P[p sp + c cp] Q[q sq + c cq].
// ---------------------------------------------------------------------------

struct NarrowArgs {
  const char *p, *q;
  const int64_t* offsets;
  char* out;
  int64_t rows, sp, cp, sq, cq, q_group, height, width;  // q_group: Q's elements a group
  int64_t length;                                        // contracted, of narrow_rows
  int groups;
};

template <class C>
__device__ inline float narrow_dot(const char* p, const char* q, const NarrowArgs& a, int64_t p0, int64_t q0,
                                   int64_t n) {
  float sum = 0.0f;
  for (int64_t c = threadIdx.x & 63; c < n; c += 64) {
    sum = __builtin_fmaf(C::load1(p, p0 + c * a.cp), C::load1(q, q0 + c * a.cq), sum);
  }
  return bits_f32(wave_allreduce(f32_bits(sum), AddF32{}));
}

// out [rows][width]: row r of group e.
template <class C>
__global__ __launch_bounds__(256) void narrow_rows(NarrowArgs a) {
  const int64_t total = a.rows * a.width;
  for (int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); i < total; i += (int64_t)gridDim.x * 4) {
    const int64_t r = i / a.width, col = i - r * a.width;
    int lo = 0, hi = a.groups + 1;  // offsets[lo - 1] <= r < offsets[hi], of those that are in order
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (a.offsets[mid] <= r) {
        lo = mid + 1;
      } else {
        hi = mid;
      }
    }
    const bool in = lo >= 1 && lo <= a.groups;
    const float v = in ? narrow_dot<C>(a.p, a.q, a, r * a.sp, (lo - 1) * a.q_group + col * a.sq, a.length) : 0.0f;
    if ((threadIdx.x & 63) == 0) C::store1(a.out, i, v);
  }
}

// out [groups][height][width]: sums over the group's rows.
template <class C>
__global__ __launch_bounds__(256) void narrow_weights(NarrowArgs a) {
  const int64_t each = a.height * a.width, total = a.groups * each;
  for (int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); i < total; i += (int64_t)gridDim.x * 4) {
    const int64_t e = i / each, h = (i - e * each) / a.width, col = i - e * each - h * a.width;
    const int64_t first = clamp_row(a.offsets[e], a.rows), end = clamp_row(a.offsets[e + 1], a.rows);
    const float v = narrow_dot<C>(a.p, a.q, a, first * a.cp + h * a.sp, first * a.cq + col * a.sq, end - first);
    if ((threadIdx.x & 63) == 0) C::store1(a.out, i, v);
  }
}

// Rows of sums of nothing.
template <class C>
__global__ __launch_bounds__(256) void zero_rows(char* __restrict__ out, int64_t elements) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < elements; i += (int64_t)gridDim.x * 256) {
    C::store1(out, i, 0.0f);
  }
}
template <class C>
int32_t launch_zero_rows(void* out, int64_t elements, hipStream_t st) {
  if (out == nullptr) return (int32_t)hipSuccess;
  zero_rows<C><<<flat_grid(elements, 256, 65536), 256, 0, st>>>(static_cast<char*>(out), elements);
  return launch_status();
}

inline unsigned narrow_grid(int64_t elements) {
  return (unsigned)(elements < 4 * 65536 ? (elements + 3) / 4 : 65536);
}

// launch(first, count) for all of `tiles` workgroups of `threads`: a launch has fewer than
// 2^32 threads, and takes a multiple of 8 tiles so that each keeps its XCD. No operands that
// a card holds make 2^31 tiles.
template <class Launch>
int32_t launch_tiles(int64_t tiles, int threads, Launch&& launch) {
  if (tiles > INT32_MAX) return (int32_t)hipErrorInvalidValue;
  const int64_t most = (int64_t(1) << 32) / threads - 8;
  for (int64_t first = 0; first < tiles; first += most) {
    launch((int)first, (unsigned)(tiles - first < most ? tiles - first : most));
    const int32_t status = launch_status();
    if (status != (int32_t)hipSuccess) return status;
  }
  return (int32_t)hipSuccess;
}

// The grid of `kernel`, whose workgroups of `threads` own BP rows and BQ columns.
template <int BP, int BQ>
int32_t launch_rows_grid(void (*kernel)(RowsArgs), int threads, RowsArgs a, hipStream_t st) {
  const int64_t edges = a.offsets == nullptr ? 1 : a.groups + 2;  // each group ends inside one tile at most
  int64_t most = (a.rows + edges * (BP - 1)) / BP;
  most = most < a.rows ? most : a.rows;
  const int64_t tiles_q = ((int64_t)a.cols + BQ - 1) / BQ;
  a.most = (int)most;
  a.tiles_q = (int)tiles_q;
  return launch_tiles(most * tiles_q, threads, [&](int first, unsigned count) {
    a.first = first;
    kernel<<<count, threads, 0, st>>>(a);
  });
}

template <class T, class C, bool QROWS, int WP, int WQ, int FP, int FQ, bool DIRECT, bool ONCE = false>
int32_t launch_rows(const RowsArgs& a, hipStream_t st) {
  return launch_rows_grid<WP * FP * 16, WQ * FQ * 16>(rows_product<T, C, QROWS, WP, WQ, FP, FQ, DIRECT, ONCE>,
                                                      WP * WQ * 64, a, st);
}

template <class T, class C, int FP, int FQ, int NW, int DEPTH>
int32_t launch_stream(const RowsArgs& a, hipStream_t st) {
  return launch_rows_grid<FP * 16, FQ * 16>(rows_stream<T, C, FP, FQ, NW, DEPTH>, NW * 64, a, st);
}

// Tiles of 256 x 256, of which a SIMD's one wave reads a quarter less from LDS for a
// product, pay where they are filled and enough for the 256 CUs. bf16, us, forward and input
// gradient, in brackets 128 x 128: 8 groups of 1024 rows, 14336 x 4096 781 and 882 (1057 and
// 1138), of 128 rows 196 and 279 (238 and 296), of 64 rows 207 and 242 (187 and 197); 64
// groups of 128 rows, 1408 x 2048 116 and 95 (110 and 97), of 160 rows 119 and 104 (118 and
// 110), of 256 rows 125 and 110 (141 and 138); 160 of 128 rows, 1536 x 2048 232 and 230 (221
// and 233), of 160 rows 252 and 252 (299 and 305).
// The group sizes are not known here: groups / 2 stands for one cut tile a group, half
// filled. Of equal groups that a tile holds there are fewer tiles, and where those are
// fewer than the CUs this rule loses: 16 groups, 2048 x 2048, 128 tiles, 192 rows 40 and 41 (31
// and 31), 256 rows 42 and 43 (35 and 35); 8 of 192 rows, 4096 x 4096, 128 tiles 83 and 82 (72
// and 70); and so does half a round too many: 32 of 320 rows, 1408 x 2048, 384 tiles 81 and 85
// (73 and 74).
template <class T>
inline bool wide_tiles(const RowsArgs& a) {
  return T::kAccumulates && a.rows >= 128 * (int64_t)a.groups &&
         (a.rows / 256 + a.groups / 2) * ((a.cols + 255) / 256) >= 150;
}

// Tiles of 128 x 128, or of 64 x 64 where there would be fewer than 192 of those for the
// 256 CUs (bf16, us, 128 against 64: 8 groups of 64 rows, 2048 x 2048, 144 tiles 31.5
// against 28.4; 16 of 128, 2048 x 1024, 200 tiles 32.9 against 34.7), and always for fp32,
// whose products take the matrix cores 16 times as long (13 groups of 77 rows, 1003 x 777:
// 70.6 against 40.7; 4096 rows, 4096 x 4096: 955 against 980).
template <class T>
inline bool middle_tiles(const RowsArgs& a) {
  return T::kBytes != 4 && (a.rows / 128 + a.groups / 2 + 1) * ((a.cols + 127) / 128) >= 192;
}
template <class T, class C, bool QROWS, bool WHOLE>
int32_t launch_rows_small(const RowsArgs& a, hipStream_t st) {
  if constexpr (T::kBytes != 4) {
    if (middle_tiles<T>(a)) {
      // Groups that fill one tile on average: their weights are read once, past the caches and
      // group after group (160 groups of 77 rows, 1536 x 2048: 184 us against 203 through the
      // caches; 64 groups of 128 rows, 1408 x 2048: 102 against 110, of 160 rows 163 against 118).
      // It loses where one group has most of the rows (12161 of those 12320: 278 against 238).
      if constexpr (WHOLE) {
        if (a.rows <= 96 * (int64_t)a.groups) return launch_rows<T, C, QROWS, 2, 2, 4, 4, true, true>(a, st);
      }
      return launch_rows<T, C, QROWS, 2, 2, 4, 4, WHOLE>(a, st);
    }
  }
  return launch_rows<T, C, QROWS, 2, 2, 2, 2, WHOLE>(a, st);
}

// Which kernel, for weights that are rows of the contracted index. The streams of few rows read
// the weights once for each 16 or 32 rows, so they are for groups that mostly have no more:
// up to half of that on average, or all of it if there is one group; and the longer one also
// where tiles are few. bf16, us, streams of 16 rows, of 32, and 128 x 128 tiles: 8 groups of 2
// rows, 14336 x 4096 121, 123, 149, of 8 rows 150, 153, 163, of 16 rows 208, 171, 152, of 32
// rows 315, 243, 158; 64 groups of 8 rows, 1408 x 2048 60, 70, 85, of 16 rows 77, 75, 83, of 24
// rows 97, 84, 84; one of 32 rows, 4096 x 4096 11, 14, 49, 14336 x 4096 33, 26, 51. One group
// with most of the rows takes the streams longer, and the tiles hardly less then (449 of 512 rows
// on 64 groups: 74 and 93; 57 of 64 on 8 of 14336 x 4096: 169 and 164). Two fragments
// of columns a workgroup, or one where that leaves CUs without (one group of 8 rows,
// 4096 x 4096 10.7 and 9.8; 64 of 8, 1408 x 2048 60 and 65).
template <class T, class C, bool WHOLE>
int32_t launch_rows_by_size(const RowsArgs& a, hipStream_t st) {
  const bool one = a.groups == 1;
  if (a.rows <= (one ? 16 : 8) * (int64_t)a.groups) {
    const int64_t tiles = a.rows < a.groups ? a.rows : a.groups;
    if (tiles * a.cols >= 256 * 32) return launch_stream<T, C, 1, 2, 4, WHOLE ? 2 : 0>(a, st);
    return launch_stream<T, C, 1, 1, 4, WHOLE ? 2 : 0>(a, st);
  }
  if (a.rows <= (one || !middle_tiles<T>(a) ? 32 : 16) * (int64_t)a.groups) {
    return launch_stream<T, C, 2, 2, 4, WHOLE ? 2 : 0>(a, st);
  }
  if constexpr (WHOLE && T::kAccumulates) {
    if (wide_tiles<T>(a)) return launch_rows<T, C, true, 2, 2, 8, 8, true>(a, st);
  }
  return launch_rows_small<T, C, true, WHOLE>(a, st);
}

// Sizes every kernel here accepts: 32-bit row counts and columns, rows that 32-bit
// offsets reach from a tile's base.
inline bool sizes_ok(int64_t rows, int64_t groups, int64_t n_bytes, int64_t k_bytes) {
  return rows >= 0 && rows <= INT32_MAX && groups >= 1 && groups <= kMaxGroups && n_bytes <= kMaxRowLength &&
         k_bytes <= kMaxRowLength;
}

}  // namespace cck

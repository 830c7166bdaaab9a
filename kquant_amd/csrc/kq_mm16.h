// Matrix products of 16-bit operands (bf16 or fp16) with fp32 accumulation, and
// of 8-bit integers with int32 accumulation, the core shared by the grouped
// products, the head loss and the int8 linear:
//
//   D[m][n] = sum over c of A(m, c) B(n, c)
//
// either operand stored along the contraction (row m holds consecutive c) or
// across it (row c holds consecutive m), so a product, both of its gradients
// and the ragged contractions of a weight gradient are one kernel body.
//
// Tile 256 x 256, contraction step 64, four waves of one per SIMD with 128 x
// 128 of the tile each (16 accumulators of 32 x 32, 256 registers).  What
// bounds it is the MFMA issue of that one wave: a step is 64
// v_mfma_f32_32x32x16 (2048 cycles), while LDS moves 128 KiB of fragment reads
// and 64 KiB of new operands for it (1536 cycles).  So everything else has a
// fixed place between two MFMAs (sched_barrier pins it):
//  * operands go HBM -> LDS by 16-byte direct loads, a step's share of one
//    operand a slab of 32 KiB, and all of LDS is five slabs: A and B of the step
//    in use and of the next one, and one operand (the leading one) of the step after.  A slab is whole
//    128-byte lines of rows (contraction-major) or 512-byte runs of 64
//    contraction rows (the other form), XOR-swizzled so that the lanes of a read
//    fall on distinct banks.
//  * a step's fragments are read one step ahead: block b of 16 MFMAs (k16
//    block b) reads the fragments of k16 block (b + 3) % 4, of this step in
//    block 0 and of the next one after it.  Operands across the contraction
//    are read transposed (ds_read_b64_tr_b16).
//  * one barrier a step, after block 0: every wave then holds all of the
//    current slabs in registers, so both are free.  The following operand of the step
//    after next is loaded in block 1, the leading one of the step after that in blocks 2 and 3: a direct
//    load takes 16 cycles of the CU's address unit, so 64 of them in one block
//    of 512 cycles held its MFMAs up (two stages of both operands, all loads in
//    block 1: 3325 cycles a step at 4096 x 12288 x 7168).
//  * a resource is rebased every step, and ends with the operand's last valid
//    row and column: rows past a ragged group or a matrix read as zero without
//    touching memory, and offsets stay below 2^31 whatever the matrix's size.
// Row tiles of at most 128 rows (the ragged end of a group) run as four waves
// side by side over the columns, 32 NB rows x 64 columns each, so rows that
// are not there cost no MFMA beyond the next 32, 64 or 128; narrow column tiles
// run as four waves down the rows.
//
// The kernels are persistent: a problem P numbers its tiles, worker w takes
// w, w + G, ... with the workers of one XCD numbered consecutively, so the 32
// tiles an XCD runs together share operand rows in its L2; the loads run on
// across tile boundaries.
#pragma once

#include <type_traits>

#include "kq_common.h"
#include "kq_dma.h"

namespace kq {
namespace mm16 {

constexpr int BM = 256, BN = 256, BK = 64, THREADS = 256;
constexpr int SLAB = 256 * BK * 2;     // one operand of a step
constexpr int SLOTS = 5;               // slabs in LDS
constexpr int LDS_BYTES = SLOTS * SLAB;
constexpr int LOADS = 8;               // direct loads per wave and slab
constexpr int GROUP_M = 4;             // row tiles per group of the tile order
constexpr uint32_t OUT_OF_RANGE = 0x80000000u;
constexpr int64_t MAX_LD = 1 << 22;    // elements: 256 rows stay below OUT_OF_RANGE

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4_t lds_s16x4_t;
typedef __attribute__((address_space(3))) u32x4_t lds_u32x4_t;

// One operand of a tile; all of it the same in every lane.
struct Operand {
  const char* base;  // the tile's first element at contraction index 0
  uint32_t ld;       // bytes between rows
  int rows;          // contraction-major: valid rows of the tile
  uint32_t width;    // across: valid bytes of a row from base
};

struct Tile {
  Operand a, b;
  int kc;    // contraction length (0 gives zeros)
  int rows;  // rows of the tile that are stored
  int cols;  // and columns
  bool once = false;  // b (the leading operand) is read for this row of tiles alone, from memory
};

// The same in every lane, in scalar registers.
__device__ __forceinline__ void make_scalar(Operand& o) {
  const uint64_t a = reinterpret_cast<uint64_t>(o.base);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)a);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32));
  o.base = reinterpret_cast<const char*>((uint64_t)hi << 32 | lo);
  o.ld = (uint32_t)__builtin_amdgcn_readfirstlane((int)o.ld);
  o.rows = __builtin_amdgcn_readfirstlane(o.rows);
  o.width = (uint32_t)__builtin_amdgcn_readfirstlane((int)o.width);
}

// Tile tl of an mtiles x ntiles grid, in groups of GROUP_M row tiles.
__device__ __forceinline__ void tile_mn(int tl, int mtiles, int ntiles, int& mt, int& nt) {
  const int per = GROUP_M * ntiles, g = tl / per, rem = tl - g * per;
  const int gsz = min(GROUP_M, mtiles - g * GROUP_M);
  mt = g * GROUP_M + rem % gsz;
  nt = rem / gsz;
}

__device__ __forceinline__ int steps_of(int kc) { return kc > BK ? (kc + BK - 1) / BK : 1; }

// This lane's LDS offsets of the fragments of NB 32-row blocks from row0 (a
// multiple of 64).
template <bool ACROSS, int NB>
struct Reader {
  uint32_t at[4];  // ACROSS: by block; else by k16 block

  __device__ __forceinline__ void set(int row0, int lane) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (ACROSS) {
        // 16-lane group g reads features 16 (g % 2) of block q and contraction
        // rows 8 (g / 2) + [0, 8); its lane s points at row s / 4 and features 4 (s % 4)
        const int g = lane >> 4, s = lane & 15, f = row0 + 32 * q + 16 * (g & 1) + 4 * (s & 3);
        at[q] = (uint32_t)((8 * (g >> 1) + (s >> 2)) * 512 + (((f >> 3) ^ (4 * (s >> 2))) << 4) + (f & 7) * 2);
      } else {
        const int row = row0 + (lane & 31);
        at[q] = (uint32_t)(row * 128 + 16 * ((2 * q + (lane >> 5)) ^ ((row >> 1) & 7)));
      }
    }
  }
  // rows row0 + 32 i + lane % 32, contraction 16 kk + 8 (lane / 32) + [0, 8) of the slab
  __device__ __forceinline__ u32x4_t read(uint32_t slab, int kk, int i) const {
    if (ACROSS) {
      const uint32_t p = slab + at[i] + (uint32_t)(kk * 16 * 512);
      const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(uintptr_t)p);
      const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(uintptr_t)(p + 4 * 512));
      return __builtin_bit_cast(u32x4_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    return *(const lds_u32x4_t*)(uintptr_t)(slab + at[kk] + (uint32_t)(i * 32 * 128));
  }
};

// What the 16-byte fragments hold.  Of 8-bit integers (I8) a pair counts as one
// element in every index and length here, and the accumulators' registers hold
// int32 bits: the same bytes and the same cycles for twice the products.
enum { BF16 = 0, F16 = 1, I8 = 2 };
typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x16_t __attribute__((ext_vector_type(16)));

template <int KIND>
__device__ __forceinline__ float16_t mfma(u32x4_t a, u32x4_t b, float16_t c) {
  if (KIND == I8)
    return __builtin_bit_cast(float16_t, __builtin_amdgcn_mfma_i32_32x32x32_i8(
                                             __builtin_bit_cast(i32x4_t, a), __builtin_bit_cast(i32x4_t, b),
                                             __builtin_bit_cast(i32x16_t, c), 0, 0, 0));
  if (KIND == F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0,
                                                  0, 0);
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0,
                                                 0, 0);
}

// Keeps block row i of the accumulators where the MFMAs left them until here:
// moved to other registers all at once after the K loop they would not fit, and
// a spill's wait for memory would stand in the loop.
template <int NB, int WN>
__device__ __forceinline__ void in_place(float16_t (&acc)[NB][WN], int i) {
#pragma unroll
  for (int j = 0; j < WN; ++j) asm volatile("" : "+a"(acc[i][j]));
}

// The elements of a wave's blocks, f(row, column, value) for rows below `rows`
// and columns below `cols` of the tile.  The row is made opaque, so that the
// offsets of the elements are not kept (and spilled) from tile to tile.
template <int NB, int WN, class F>
__device__ __forceinline__ void each(int rows, int cols, int wm, int wn, float16_t (&acc)[NB][WN], int lane, F&& f) {
  int row = wm + 4 * (lane >> 5);
  const int col = wn + (lane & 31);
  asm volatile("" : "+v"(row));
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    in_place(acc, i);
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int at = row + 32 * i + 8 * (r >> 2) + (r & 3);
      if (at < rows) {
#pragma unroll
        for (int j = 0; j < WN; ++j)
          if (col + 32 * j < cols) f(at, col + 32 * j, acc[i][j][r]);
      }
    }
  }
}

// Two 16-bit values of a row pair, rounded to nearest even.
template <bool F16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  return F16 ? f32x2_to_f16x2_bits(lo, hi) : f32x2_to_bf16x2_bits(lo, hi);
}

// The value of lane ^ 4.
__device__ __forceinline__ uint32_t other_quad(uint32_t v) {
  const int up = __builtin_amdgcn_update_dpp(0, (int)v, 0x104, 0xf, 0x5, true);     // even quads: lane + 4
  return (uint32_t)__builtin_amdgcn_update_dpp(up, (int)v, 0x114, 0xf, 0xa, true);  // odd quads: lane - 4
}

// Four rows (elements 4 g .. 4 g + 3 as f(i, j, r, value)) of the columns of
// WN blocks, exchanged over the lane's quad for four columns of one row, in 16
// bits.  One wave runs on a SIMD, so an instruction that waits for the one
// before it costs the wave its latency: each step of the exchange is taken for
// all blocks before the next.
template <int NB, int WN, bool F16, class F>
__device__ __forceinline__ void quad_rows(const float16_t (&acc)[NB][WN], int i, int g, u32x2_t (&v)[WN], F&& f) {
  const int t = (int)threadIdx.x & 3;
  const uint32_t sel = t & 1 ? 0x03020706u : 0x05040100u;  // as quad_transpose16
  uint32_t w0[WN], w1[WN], p0[WN], p1[WN], got[WN];
#pragma unroll
  for (int j = 0; j < WN; ++j) {
    const int r = 4 * g;
    w0[j] = pack16<F16>(f(i, j, r, acc[i][j][r]), f(i, j, r + 1, acc[i][j][r + 1]));
    w1[j] = pack16<F16>(f(i, j, r + 2, acc[i][j][r + 2]), f(i, j, r + 3, acc[i][j][r + 3]));
  }
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int j = 0; j < WN; ++j) {
    p0[j] = (uint32_t)__builtin_amdgcn_mov_dpp((int)w0[j], 0xb1, 0xf, 0xf, true);  // lane ^ 1
    p1[j] = (uint32_t)__builtin_amdgcn_mov_dpp((int)w1[j], 0xb1, 0xf, 0xf, true);
  }
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int j = 0; j < WN; ++j) {
    w0[j] = __builtin_amdgcn_perm(p0[j], w0[j], sel);
    w1[j] = __builtin_amdgcn_perm(p1[j], w1[j], sel);
  }
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int j = 0; j < WN; ++j) got[j] = t & 2 ? w0[j] : w1[j];
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int j = 0; j < WN; ++j) got[j] = (uint32_t)__builtin_amdgcn_mov_dpp((int)got[j], 0x4e, 0xf, 0xf, true);  // lane ^ 2
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int j = 0; j < WN; ++j) {
    v[j][0] = t & 2 ? got[j] : w0[j];
    v[j][1] = t & 2 ? w1[j] : got[j];
  }
}

// The same exchanged over two quads, for pairs of blocks: eight columns of one
// row, of the first block in the even quad and of the second in the odd one.
template <int NB, int WN, bool F16, class F>
__device__ __forceinline__ void eight_columns(const float16_t (&acc)[NB][WN], int i, int g, u32x4_t (&q)[WN / 2], F&& f) {
  const bool odd = threadIdx.x & 4;
  u32x2_t v[WN];
  quad_rows<NB, WN, F16>(acc, i, g, v, f);
  __builtin_amdgcn_sched_barrier(0);
  uint32_t x0[WN / 2], x1[WN / 2];
#pragma unroll
  for (int j = 0; j < WN; j += 2) {
    x0[j / 2] = odd ? v[j][0] : v[j + 1][0];
    x1[j / 2] = odd ? v[j][1] : v[j + 1][1];
  }
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int j = 0; j < WN / 2; ++j) {
    x0[j] = other_quad(x0[j]);
    x1[j] = other_quad(x1[j]);
  }
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int j = 0; j < WN; j += 2) {
    q[j / 2][0] = odd ? x0[j / 2] : v[j][0];
    q[j / 2][1] = odd ? x1[j / 2] : v[j][1];
    q[j / 2][2] = odd ? v[j + 1][0] : x0[j / 2];
    q[j / 2][3] = odd ? v[j + 1][1] : x1[j / 2];
  }
}

// Stores a wave's blocks in 16 bits: rows below `rows`, columns below `cols` (a
// multiple of 8) of the tile, f(i, j, r, v) the value stored for element r of
// block (i, j), v the accumulated one; address(row) is the 16-byte aligned
// address of a row's column 0 (asked for rows below `rows` only).
// A store instruction takes the CU's memory path some 8 cycles for each line it
// touches, so it should fill them: a lane's four rows of one column are
// exchanged over two quads for eight columns of one row, of which 8 lanes make
// a 128-byte line.  Results are larger than an XCD's L2 and read from another
// one: nontemporal.  48 weight gradients of 7168 x 2048, 64 rows each: 461 us
// with 8 bytes a lane, 402 nontemporal, 290 with 16 bytes (1.41 GB).
template <int NB, int WN, bool F16, class At, class F>
__device__ __forceinline__ void store16(At&& address, int rows, int cols, int wm, int wn, float16_t (&acc)[NB][WN],
                                        int lane, F&& f) {
  int row = wm + 4 * (lane >> 5) + (lane & 3), col = wn + (lane & 28);
  if (WN > 1 && (lane & 4)) col += 28;  // the second block, from 4 columns to the left
  asm volatile("" : "+v"(row), "+v"(col));  // the elements' offsets are not kept (and spilled) from tile to tile
  auto block_rows = [&](auto whole) {
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      in_place(acc, i);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int at = row + 32 * i + 8 * g;
        char* p = address(whole.value ? at : min(at, rows - 1)) + 2 * (int64_t)col;
        if constexpr (WN > 1) {
          u32x4_t q[WN / 2];
          eight_columns<NB, WN, F16>(acc, i, g, q, f);
#pragma unroll
          for (int j = 0; j < WN / 2; ++j)
            if (whole.value || (at < rows && col + 64 * j < cols))
              __builtin_nontemporal_store(q[j], reinterpret_cast<u32x4_t*>(p + 128 * j));
        } else {
          u32x2_t v[WN];
          quad_rows<NB, WN, F16>(acc, i, g, v, f);
          if (at < rows && col < cols) __builtin_nontemporal_store(v[0], reinterpret_cast<u32x2_t*>(p));
        }
        if (!whole.value) __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  if constexpr (NB * WN == 16) {
    if (rows >= BM && cols >= BN) {  // without masks and their branches
      block_rows(std::true_type{});
      return;
    }
  }
  block_rows(std::false_type{});
}

// One operand's loads, slab after slab, across this worker's tiles.  The
// resource of the next slab is made when the last one's loads are out, in a few
// scalar instructions: 64 contraction indices on, and only a tile's last slab
// is shorter.
template <bool ACROSS>
struct Side {
  dma::i32x4_t r;
  int i, k, kc;       // tile (of this worker's), contraction index of the next slab, the tile's contraction length
  uint32_t inc;       // bytes from slab to slab
  uint32_t ld, rows;  // the tile's row stride and valid rows (contraction-major)
  uint32_t width;     // its valid bytes of a row (across)
  uint32_t off, at, step;  // this lane's offset in a slab, in this slab, and from load to load
  int col;            // contraction-major: this lane's first contraction index in a slab
  bool once;          // the tile's operand is read once

  // what the slab at k ends with: rows and columns past it read as zero
  __device__ __forceinline__ void limit() {
    const int left = kc - k, n = left < BK ? left : BK;
    if (ACROSS) {
      r[2] = n > 0 ? (int)((uint32_t)(n - 1) * ld + width) : 0;
    } else {
      r[2] = n > 0 && rows > 0 ? (int)((rows - 1) * ld + 2u * (uint32_t)n) : 0;
      at = col < left ? off : OUT_OF_RANGE;
    }
  }
  template <class P, class Pick>
  __device__ __forceinline__ void set(const P& p, int tiles, int lw, int lane, Pick&& pick) {
    k = 0;
    once = false;
    kc = 0;  // loads past the last tile read zeros and touch nothing
    if (i < tiles) {
      const Tile t = p.tile(i);
      Operand o = pick(t);
      make_scalar(o);
      kc = __builtin_amdgcn_readfirstlane(t.kc);
      once = __builtin_amdgcn_readfirstlane((int)t.once) != 0;
      r = dma::make_rsrc(o.base, 0);
      ld = o.ld;
      rows = (uint32_t)o.rows;
      width = o.width;
      inc = ACROSS ? BK * o.ld : BK * 2;
      if (ACROSS) {
        const int row = 2 * lw + (lane >> 5);
        off = at = (uint32_t)row * o.ld + (uint32_t)(((lane & 31) ^ (4 * (row & 3))) * 16);
        step = 8 * o.ld;
      } else {
        const int row = 8 * lw + (lane >> 3), ch = (lane & 7) ^ ((row >> 1) & 7);
        off = (uint32_t)row * o.ld + (uint32_t)(ch * 16);
        step = 32 * o.ld;
        col = 8 * ch;
      }
    }
    limit();
  }
  // load u (0..7) of the slab at k into LDS slot base `slot`: 1 KiB at (4 u + lw) * 1024
  __device__ __forceinline__ void issue(int u, uint32_t slot, int lw) const {
    dma::load_to_lds16(r, at + (uint32_t)u * step, slot + (uint32_t)((4 * u + lw) * 1024));
  }
  __device__ __forceinline__ void issue_once(int u, uint32_t slot, int lw) const {
    dma::load_to_lds16_nt(r, at + (uint32_t)u * step, slot + (uint32_t)((4 * u + lw) * 1024));
  }
  // loads that hold a valid row (contraction-major; the others write zeros that only rows past the tile read)
  __device__ __forceinline__ int needed() const { return ACROSS ? LOADS : (int)(rows + 31) / 32; }
  // The next slab: of this tile in straight-line scalar code; what the tile's last slab and its end need is out of the
  // way (a taken branch stops the one wave's issue: 4096 x 12288 x 7168 forward / dx / dw 521 / 575 / 590 us with it in
  // line, 505 / 564 / 577 so).  False at the end.
  __device__ __forceinline__ bool next() {
    k += BK;
    const uint32_t lo = (uint32_t)r[0] + inc;
    r[1] += lo < inc ? 1 : 0;
    r[0] = (int)lo;
    if (__builtin_expect(kc - k < BK, 0)) {
      if (k >= kc) return false;
      limit();
    }
    return true;
  }
};

enum { WHOLE = 0, SMALL_ROWS = 1, SMALL_COLS = 2 };  // which tiles may be narrow

// The tiles of problem P, worker by worker.  P has
//   int tiles()          this worker's number of them
//   Tile tile(int i)     its i-th
//   epilogue<NB, WN>(const Tile&, int i, int wm, int wn, float16_t (&acc)[NB][WN], int lane)
// with element r of acc[a][b] at row wm + 32 a + 8 (r / 4) + 4 (lane / 32) + r % 4,
// column wn + 32 b + lane % 32 of the tile.
//
// LEAD_B: B's loads run a step further ahead than A's, not A's than B's: for
// the operand that comes from memory rather than from a cache.  (Narrow tiles'
// steps are shorter than memory's latency: 64 rows in 48 groups, 4096 x 7168,
// forward 443 us with A's ahead, 404 with B's.)  ONCE: narrow tiles load a B that
// is read for them alone nontemporally: 384 -> 349 us.
// Not B that others read too or that may still be in a cache: 12 groups of
// 1416 x 1032 again and again, 21 us a call and 29 so.
template <bool AA, bool BA, int KIND, int NARROW, bool LEAD_B, bool ONCE, class P>
struct Core {
  const P& p;
  uint32_t lds0;
  int lane, lw, tiles;
  Side<AA> sa;
  Side<BA> sb;
  int cl, cf;  // slots of the slabs in use: the leading operand's and the other's
  // Every wave has issued STORES stores or more since the loads of the next step's slabs.  All are waited for in the
  // order of issue, and LOADS loads of a later slab stand between: with STORES + LOADS outstanding the slabs have
  // landed, and the stores need not have.
  bool stored;
  static constexpr int STORES = 32;

  __device__ __forceinline__ Core(const P& prob, unsigned char* l) : p(prob) {
    lane = threadIdx.x & 63;
    lw = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    lds0 = dma::lds_offset_of(l);
  }
  static __device__ __forceinline__ int after(int slot) { return slot >= SLOTS - 2 ? slot - (SLOTS - 2) : slot + 2; }
  __device__ __forceinline__ uint32_t slot(int c) const { return lds0 + (uint32_t)(c * SLAB); }
  __device__ __forceinline__ void set_a() { sa.set(p, tiles, lw, lane, [](const Tile& t) { return t.a; }); }
  __device__ __forceinline__ void set_b() { sb.set(p, tiles, lw, lane, [](const Tile& t) { return t.b; }); }
  __device__ __forceinline__ void next_a() {
    if (__builtin_expect(!sa.next(), 0)) {
      ++sa.i;
      set_a();
    }
  }
  __device__ __forceinline__ void next_b() {
    if (__builtin_expect(!sb.next(), 0)) {
      ++sb.i;
      set_b();
    }
  }

  __device__ __forceinline__ void lead_issue(int u, uint32_t to) {
    if (LEAD_B) sb.issue(u, to, lw);
    else sa.issue(u, to, lw);
  }
  __device__ __forceinline__ void lead_next() {
    if (LEAD_B) next_b();
    else next_a();
  }
  __device__ __forceinline__ void follow_issue(int u, uint32_t to) {
    if (LEAD_B) sa.issue(u, to, lw);
    else sb.issue(u, to, lw);
  }
  __device__ __forceinline__ void follow_next() {
    if (LEAD_B) next_a();
    else next_b();
  }

  // Wave tile of NB x WN blocks at (wm, wn): this item's steps, then its epilogue.
  template <int NB, int WN>
  __device__ __forceinline__ void item(const Tile& tl, int it, int wm, int wn) {
    Reader<AA, NB> fa;
    Reader<BA, WN> fb;
    int l = lane;
    asm volatile("" : "+v"(l));  // offsets are made per tile, not kept for every form of it
    fa.set(wm, l);
    fb.set(wn, l);
    u32x4_t a[4][NB], b[4][WN];
    float16_t acc[NB][WN];
    // fragment f of k16 block kk: 0..NB-1 of A, then B
    auto read_one = [&](uint32_t lead, uint32_t follow, int kk, int f) {
      if (f < NB) a[kk][f] = fa.read(LEAD_B ? follow : lead, kk, f);
      else b[kk][f - NB] = fb.read(LEAD_B ? lead : follow, kk, f - NB);
    };
    const int steps = steps_of(tl.kc);
    // this item's first slabs have landed: in run() or at the last barrier of the item before
#pragma unroll
    for (int kk = 0; kk < 3; ++kk)
#pragma unroll
      for (int f = 0; f < NB + WN; ++f) read_one(slot(cl), slot(cf), kk, f);
    __builtin_amdgcn_sched_barrier(0);  // the accumulators are cleared while these are on their way
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int j = 0; j < WN; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
    constexpr int NM = NB * WN;  // MFMAs of a k16 block
    for (int s = 0; s < steps; ++s) {
      // Narrow tiles: loads of the following operand's rows that are there.  The barrier below counts the leading
      // operand's alone, which are younger.
      const int few = LEAD_B ? sa.needed() : sb.needed();
      const uint32_t lcur = slot(cl), fcur = slot(cf), lnxt = slot(after(cl)), fnxt = slot(after(cf));
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
#pragma unroll
        for (int m = 0; m < NM; ++m) {
          const int i = m / WN, j = m % WN;
          acc[i][j] = mfma<KIND>(a[kk][i], b[kk][j], acc[i][j]);
          // block 0 reads in its first half, so that nothing is in flight at the barrier
          constexpr int HALF = NM > 1 ? NM / 2 : 1;
          const int rn = kk == 0 ? HALF : NM;
#pragma unroll
          for (int f = 0; f < NB + WN; ++f)
            if (f * rn / (NB + WN) == m)
              read_one(kk == 0 ? lcur : lnxt, kk == 0 ? fcur : fnxt, (kk + 3) & 3, f);
          if (kk == 1) {  // the following operand of the step after next, into the leading one's slot
#pragma unroll
            for (int u = m * LOADS / NM; u < (m + 1) * LOADS / NM; ++u)
              if (NM == 16 || u < few) follow_issue(u, lcur);
          }
          if (kk >= 2) {  // the leading operand of the step after that, into the other's slot
#pragma unroll
            for (int u = ((kk - 2) * NM + m) * LOADS / (2 * NM); u < ((kk - 2) * NM + m + 1) * LOADS / (2 * NM); ++u)
              if (ONCE && NM != 16 && sb.once) sb.issue_once(u, fcur, lw);
              else lead_issue(u, fcur);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        if (kk == 0) {
          __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): no read of the current slabs is in flight
          // the next slabs have landed, the current ones are free
          if (s == 0 && stored) dma::wait_and_barrier<LOADS + STORES>();
          else dma::wait_and_barrier<LOADS>();
          __builtin_amdgcn_sched_barrier(0);
        }
        if (kk == 1) follow_next();
        if (kk == 3) lead_next();
      }
      cl = after(cl);
      cf = after(cf);
    }
    stored = p.template epilogue<NB, WN>(tl, it, wm, wn, acc, l) && NB * WN == 16;
    // an epilogue that ends in a lane's branch must not be the tile loop's last statement: the loop would be taken
    // for one of divergent exit, and its scalars (the loads' resources) would be kept in vector registers
    __builtin_amdgcn_sched_barrier(0);
  }

  __device__ __forceinline__ void run() {
    tiles = __builtin_amdgcn_readfirstlane(p.tiles());
    if (tiles <= 0) return;
    sa.i = sb.i = 0;
    cl = 0;
    cf = 1;
    stored = false;
    set_a();
    set_b();
#pragma unroll
    for (int q = 0; q < SLOTS; ++q) {  // leading, following, leading, following, leading
#pragma unroll
      for (int u = 0; u < LOADS; ++u) {
        if (q & 1) follow_issue(u, slot(q));
        else lead_issue(u, slot(q));
      }
      if (q & 1) follow_next();
      else lead_next();
    }
    dma::wait_and_barrier<(SLOTS - 2) * LOADS>();
    for (int i = 0; i < tiles; ++i) {
      Tile tl = p.tile(i);
      tl.kc = __builtin_amdgcn_readfirstlane(tl.kc);
      tl.rows = __builtin_amdgcn_readfirstlane(tl.rows);
      tl.cols = __builtin_amdgcn_readfirstlane(tl.cols);
      if constexpr (NARROW == SMALL_ROWS) {
        if (tl.rows <= 128) {
          if (tl.rows <= 32) item<1, 2>(tl, i, 0, 64 * lw);
          else if (tl.rows <= 64) item<2, 2>(tl, i, 0, 64 * lw);
          else if (KIND == I8 && tl.rows <= 96) item<KIND == I8 ? 3 : 4, 2>(tl, i, 0, 64 * lw);
          else item<4, 2>(tl, i, 0, 64 * lw);
          continue;
        }
      }
      if constexpr (NARROW == SMALL_COLS) {
        if (tl.cols <= 128) {
          if (tl.cols <= 32) item<2, 1>(tl, i, 64 * lw, 0);
          else if (tl.cols <= 64) item<2, 2>(tl, i, 64 * lw, 0);
          else item<2, 4>(tl, i, 64 * lw, 0);
          continue;
        }
      }
      item<4, 4>(tl, i, (lw >> 1) * 128, (lw & 1) * 128);
    }
    __builtin_amdgcn_s_waitcnt(dma::waitcnt_vm(0));  // no load may land after the workgroup ends
  }
};

// Workers of one XCD (workgroup b runs on XCD b % 8) are numbered consecutively.
__device__ __forceinline__ int worker_number() {
  return (int)(blockIdx.x % 8) * ((int)gridDim.x / 8) + (int)(blockIdx.x / 8);
}
__device__ __forceinline__ int worker_tiles(int total) {
  const int w = worker_number(), g = (int)gridDim.x;
  return total > w ? (total - w - 1) / g + 1 : 0;
}

}  // namespace mm16
}  // namespace kq

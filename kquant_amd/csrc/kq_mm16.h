// Matrix products of 16-bit operands (bf16 or fp16) with fp32 accumulation,
// the core shared by the grouped products and the head loss:
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
//  * operands go HBM -> LDS by 16-byte direct loads into two stages of 64 KiB.
//    A stage is whole 128-byte lines of rows (contraction-major) or 512-byte
//    runs of 64 contraction rows (the other form), XOR-swizzled so that the
//    lanes of a read fall on distinct banks.
//  * a step's fragments are read one step ahead: block b of 16 MFMAs (k16
//    block b) reads the fragments of k16 block (b + 3) % 4, of this step in
//    block 0 and of the next one after it.  Operands across the contraction
//    are read transposed (ds_read_b64_tr_b16).
//  * one barrier a step, after block 0: every wave then holds all of the
//    current stage in registers, so the stage is free and the loads of the
//    step after next go into it, in block 1.
//  * a resource is rebased every step, and ends with the operand's last valid
//    row and column: rows past a ragged group or a matrix read as zero without
//    touching memory, and offsets stay below 2^31 whatever the matrix's size.
// Row tiles of at most 128 rows (the ragged end of a group) run as four waves
// side by side over the columns, 32 NB rows x 64 columns each, so rows that
// are not there cost no MFMA beyond the next 32, 64 or 128.
//
// The kernels are persistent: a problem P numbers its tiles, worker w takes
// w, w + G, ... with the workers of one XCD numbered consecutively, so the 32
// tiles an XCD runs together share operand rows in its L2; the loads run on
// across tile boundaries.
#pragma once

#include "kq_common.h"
#include "kq_dma.h"

namespace kq {
namespace mm16 {

constexpr int BM = 256, BN = 256, BK = 64, THREADS = 256;
constexpr int SLAB = 256 * BK * 2;     // one operand of a stage
constexpr int STAGE = 2 * SLAB;
constexpr int LDS_BYTES = 2 * STAGE;
constexpr int LOADS = 8;               // direct loads per wave, operand and stage
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

// The direct loads of one operand: this lane's offset in a stage, and the
// resource of the stage that starts at contraction index k0.
template <bool ACROSS>
struct Loader {
  uint32_t off, step;
  int col;  // contraction-major: this lane's first contraction index in a stage

  __device__ __forceinline__ void set(const Operand& o, int lw, int lane) {
    if (ACROSS) {
      const int row = 2 * lw + (lane >> 5);
      off = (uint32_t)row * o.ld + (uint32_t)(((lane & 31) ^ (4 * (row & 3))) * 16);
      step = 8 * o.ld;
      col = 0;
    } else {
      const int row = 8 * lw + (lane >> 3), ch = (lane & 7) ^ ((row >> 1) & 7);
      off = (uint32_t)row * o.ld + (uint32_t)(ch * 16);
      step = 32 * o.ld;
      col = 8 * ch;
    }
  }
  // load u (0..7) goes to LDS offset (4 u + lw) * 1024 of the operand's slab
  __device__ __forceinline__ uint32_t offset(int u, int left) const {
    return (ACROSS || col < left ? off : OUT_OF_RANGE) + (uint32_t)u * step;
  }
  static __device__ __forceinline__ dma::i32x4_t resource(const Operand& o, int k0, int kc) {
    const int left = kc - k0;
    if (ACROSS) {
      const int rows = left < BK ? left : BK;
      return dma::make_rsrc(o.base + (int64_t)k0 * o.ld, rows > 0 ? (uint32_t)(rows - 1) * o.ld + o.width : 0u);
    }
    const int wide = left < BK ? left : BK;
    return dma::make_rsrc(o.base + 2 * (int64_t)k0,
                          o.rows > 0 && left > 0 ? (uint32_t)(o.rows - 1) * o.ld + 2u * (uint32_t)wide : 0u);
  }
};

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

template <bool F16>
__device__ __forceinline__ float16_t mfma(u32x4_t a, u32x4_t b, float16_t c) {
  if (F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0,
                                                  0, 0);
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0,
                                                 0, 0);
}

// The elements of a wave's blocks, f(row, column, value) for rows below `rows`
// and columns below `cols` of the tile.  The row is made opaque, so that the
// offsets of the elements are not kept (and spilled) from tile to tile.
template <int NB, int WN, class F>
__device__ __forceinline__ void each(int rows, int cols, int wm, int wn, const float16_t (&acc)[NB][WN], int lane,
                                     F&& f) {
  int row = wm + 4 * (lane >> 5);
  const int col = wn + (lane & 31);
  asm volatile("" : "+v"(row));
#pragma unroll
  for (int i = 0; i < NB; ++i)
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

// Two 16-bit values of a row pair, rounded to nearest even.
template <bool F16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  return F16 ? f32x2_to_f16x2_bits(lo, hi) : f32x2_to_bf16x2_bits(lo, hi);
}

// Stores a wave's blocks in 16 bits: rows below `rows`, columns below `cols` (a
// multiple of 4) of the tile, f(i, j, r) the value of element r of block (i,
// j), address(row) the 8-byte aligned address of a row's column 0 (asked for rows
// below `rows` only).  A lane holds four rows of one column and
// exchanges them with its quad for four columns of one row, in 10 instructions
// of its registers, so it stores 8 bytes: a store instruction takes as long for
// 2 bytes a lane.
template <int NB, int WN, bool F16, class At, class F>
__device__ __forceinline__ void store16(At&& address, int rows, int cols, int wm, int wn, int lane, F&& f) {
  const int t = lane & 3;
  int row = wm + 4 * (lane >> 5) + t, col = wn + (lane & 28);
  asm volatile("" : "+v"(row), "+v"(col));  // the elements' offsets are not kept (and spilled) from tile to tile
  // even lanes: the low halves of (own, partner), odd lanes: the high halves of (partner, own)
  const uint32_t sel = t & 1 ? 0x03020706u : 0x05040100u;
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int at = row + 32 * i + 8 * g;
      char* p = address(min(at, rows - 1)) + 2 * (int64_t)col;
#pragma unroll
      for (int j = 0; j < WN; ++j) {
        uint32_t q[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t own = pack16<F16>(f(i, j, 4 * g + 2 * h), f(i, j, 4 * g + 2 * h + 1));
          const uint32_t other = (uint32_t)__builtin_amdgcn_mov_dpp((int)own, 0xb1, 0xf, 0xf, true);  // lane ^ 1
          q[h] = __builtin_amdgcn_perm(other, own, sel);
        }
        const uint32_t send = t & 2 ? q[0] : q[1];
        const uint32_t got = (uint32_t)__builtin_amdgcn_mov_dpp((int)send, 0x4e, 0xf, 0xf, true);  // lane ^ 2
        u32x2_t v;
        v[0] = t & 2 ? got : q[0];
        v[1] = t & 2 ? q[1] : got;
        if (at < rows && col + 32 * j < cols) *reinterpret_cast<u32x2_t*>(p + 64 * j) = v;
      }
    }
}

// The tiles of problem P, worker by worker.  P has
//   int total()                         tiles
//   Tile tile(int t, int& hint)         tile t (hint: this caller's, 0 at first; t never falls)
//   epilogue<NB, WN>(const Tile&, int t, int hint, int wm, int wn, const float16_t (&acc)[NB][WN], int lane)
// with element r of acc[i][j] at row wm + 32 i + 8 (r / 4) + 4 (lane / 32) + r % 4,
// column wn + 32 j + lane % 32 of the tile.  SMALL: row tiles of up to 128
// rows occur.
template <bool AA, bool BA, bool F16, bool SMALL, class P>
struct Core {
  const P& p;
  uint32_t lds0;
  int lane, lw, G;
  // load side: item lt's tile and the next stage's contraction index and slot
  int lt, lk, lslot, lhint;
  Tile ld;
  Loader<AA> la;
  Loader<BA> lb;
  int cslot;  // stage in use

  __device__ __forceinline__ Core(const P& prob, unsigned char* l) : p(prob) {
    lane = threadIdx.x & 63;
    lw = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    lds0 = dma::lds_offset_of(l);
    G = gridDim.x;
  }
  __device__ __forceinline__ void set_load_tile() {
    lk = 0;
    if (lt < p.total()) {
      ld = p.tile(lt, lhint);
      make_scalar(ld.a);
      make_scalar(ld.b);
      ld.kc = __builtin_amdgcn_readfirstlane(ld.kc);
      la.set(ld.a, lw, lane);
      lb.set(ld.b, lw, lane);
    } else {
      ld.kc = 0;  // loads past the end read zeros and touch nothing
    }
  }
  // load u of the next stage: 0..7 operand A, 8..15 operand B
  __device__ __forceinline__ void issue_one(int u, const dma::i32x4_t& ra, const dma::i32x4_t& rb) {
    const uint32_t base = lds0 + (uint32_t)(lslot * STAGE);
    if (u < LOADS)
      dma::load_to_lds16(ra, la.offset(u, ld.kc - lk), base + (uint32_t)((4 * u + lw) * 1024));
    else
      dma::load_to_lds16(rb, lb.offset(u - LOADS, ld.kc - lk), base + (uint32_t)(SLAB + (4 * (u - LOADS) + lw) * 1024));
  }
  __device__ __forceinline__ void resources(dma::i32x4_t& ra, dma::i32x4_t& rb) {
    ra = Loader<AA>::resource(ld.a, lk, ld.kc);
    rb = Loader<BA>::resource(ld.b, lk, ld.kc);
  }
  __device__ __forceinline__ void advance() {
    lslot ^= 1;
    lk += BK;
    if (lk >= ld.kc) {
      lt += G;
      set_load_tile();
    }
  }
  __device__ __forceinline__ void issue_stage() {
    dma::i32x4_t ra, rb;
    resources(ra, rb);
#pragma unroll
    for (int u = 0; u < 2 * LOADS; ++u) issue_one(u, ra, rb);
    advance();
  }

  // Wave tile of NB x WN blocks at (wm, wn): this item's steps, then its epilogue.
  template <int NB, int WN>
  __device__ __forceinline__ void item(const Tile& tl, int t, int hint, int wm, int wn) {
    Reader<AA, NB> fa;
    Reader<BA, WN> fb;
    int l = lane;
    asm volatile("" : "+v"(l));  // offsets are made per tile, not kept for every form of it
    fa.set(wm, l);
    fb.set(wn, l);
    u32x4_t a[4][NB], b[4][WN];
    float16_t acc[NB][WN];
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int j = 0; j < WN; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
    // fragment f of k16 block kk: 0..NB-1 of A, then B
    auto read_one = [&](uint32_t st, int kk, int f) {
      if (f < NB) a[kk][f] = fa.read(st, kk, f);
      else b[kk][f - NB] = fb.read(st + SLAB, kk, f - NB);
    };
    const int steps = steps_of(tl.kc);
    {  // this item's first stage has landed: in run() or at the last barrier of the item before

      const uint32_t st = lds0 + (uint32_t)(cslot * STAGE);
#pragma unroll
      for (int kk = 0; kk < 3; ++kk)
#pragma unroll
        for (int f = 0; f < NB + WN; ++f) read_one(st, kk, f);
    }
    constexpr int NM = NB * WN;  // MFMAs of a k16 block
    for (int s = 0; s < steps; ++s) {
      const uint32_t cur = lds0 + (uint32_t)(cslot * STAGE), nxt = lds0 + (uint32_t)((cslot ^ 1) * STAGE);
      dma::i32x4_t ra, rb;
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
#pragma unroll
        for (int m = 0; m < NM; ++m) {
          const int i = m / WN, j = m % WN;
          acc[i][j] = mfma<F16>(a[kk][i], b[kk][j], acc[i][j]);
          // fragments of k16 block (kk + 3) % 4 and, in block 1, the loads
#pragma unroll
          for (int f = m * (NB + WN) / NM; f < (m + 1) * (NB + WN) / NM; ++f)
            read_one(kk == 0 ? cur : nxt, (kk + 3) & 3, f);
          if (kk == 1) {
#pragma unroll
            for (int u = m * 2 * LOADS / NM; u < (m + 1) * 2 * LOADS / NM; ++u) issue_one(u, ra, rb);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        if (kk == 0) {
          __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): no read of the current stage is in flight
          dma::wait_and_barrier<0>();          // the next stage has landed, the current one is free
          resources(ra, rb);
          __builtin_amdgcn_sched_barrier(0);
        }
        if (kk == 1) advance();
      }
      cslot ^= 1;
    }
    p.template epilogue<NB, WN>(tl, t, hint, wm, wn, acc, l);
  }

  __device__ __forceinline__ void run() {
    const int worker = (int)(blockIdx.x % 8) * (G / 8) + (int)(blockIdx.x / 8);
    const int total = p.total();
    if (worker >= total) return;
    lt = worker;
    lslot = cslot = 0;
    lhint = 0;
    set_load_tile();
    issue_stage();
    issue_stage();
    dma::wait_and_barrier<2 * LOADS>();
    int hint = 0;
    for (int t = worker; t < total; t += G) {
      const Tile tl = p.tile(t, hint);
      if (SMALL && tl.rows <= 128) {
        if (tl.rows <= 32) item<1, 2>(tl, t, hint, 0, 64 * lw);
        else if (tl.rows <= 64) item<2, 2>(tl, t, hint, 0, 64 * lw);
        else item<4, 2>(tl, t, hint, 0, 64 * lw);
      } else {
        item<4, 4>(tl, t, hint, (lw >> 1) * 128, (lw & 1) * 128);
      }
    }
    __builtin_amdgcn_s_waitcnt(dma::waitcnt_vm(0));  // no load may land after the workgroup ends
  }
};

}  // namespace mm16
}  // namespace kq

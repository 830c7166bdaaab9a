// The kernel of the products grouped by expert, for dense 16-bit operands and for
// 8-bit integers: how a workgroup numbers the tiles of ragged groups whose sizes
// stay on the device.
#pragma once

#include "kq_int8.h"
#include "kq_internal.h"

namespace kq {
namespace grouped {

constexpr int MAX_GROUPS = 4096;
enum { FORWARD = 0, DX = 1, DW = 2 };

struct Args {
  const char* rows_in;    // x (forward), dy (dx, dw)
  const char* other;      // w, or x (dw)
  char* out;              // y, dx, dw
  uint32_t ld_in, ld_other, ld_out;  // bytes
  const int64_t* offsets;
  int64_t rows;
  int groups, n, k;
  const float* sx = nullptr;  // int8: scales of the rows and of the weights' rows
  const float* sw = nullptr;
};

constexpr int64_t LAST_LEVEL_CACHE = 256ll << 20;
constexpr int TABLE = 4;  // 64 tiles of a worker each

// Offsets are device data: clamped to the rows there are, so that no value of
// them reads or writes outside.
__device__ __forceinline__ int64_t clamped(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : v > hi ? hi : v; }

// STREAM: the weights are more than the last-level cache holds.  KIND I8: codes,
// with k in pairs of them, and results of type OUT (KQ_DT_*).
template <int MODE, int KIND, bool STREAM, int OUT = 0>
struct Problem {
  Args g;
  int mtiles, ntiles, count;
  // lane l of entry q: this worker's tile 64 q + l
  int group_nt[TABLE], mt_of[TABLE], beg_of[TABLE], n_of[TABLE];

  __device__ __forceinline__ void range(int e, int& beg, int& n) const {
    // constant memory, so that a group that is the same in every lane takes scalar loads
    const auto* o = (const __attribute__((address_space(4))) int64_t*)g.offsets + e;
    const int64_t b = clamped(o[0], 0, g.rows);
    beg = (int)b;
    n = (int)(clamped(o[1], b, g.rows) - b);
  }
  __device__ __forceinline__ int tiles() const { return count; }

  // Tiles of a group of n rows.
  __device__ __forceinline__ int tiles_of(int n) const {
    return (MODE == DW ? mtiles : (n + mm16::BM - 1) / mm16::BM) * ntiles;
  }

  // Numbers the tiles; every thread of the workgroup calls it, before the slabs
  // use LDS.  The groups' tiles are summed in LDS, then every lane looks one of
  // the worker's tiles up, so the K loops find theirs in a register.
  __device__ __forceinline__ void setup(unsigned char* lds) {
    const int cols = MODE == FORWARD ? g.n : g.k;
    ntiles = (cols + mm16::BN - 1) / mm16::BN;
    mtiles = (g.n + mm16::BM - 1) / mm16::BM;
    int* first = reinterpret_cast<int*>(lds);  // [groups + 1]
    int* part = first + MAX_GROUPS + 1;
    const int t = threadIdx.x, per = (g.groups + mm16::THREADS - 1) / mm16::THREADS;
    const int e0 = min(t * per, g.groups), e1 = min(e0 + per, g.groups);
    // Offsets that decrease make groups overlap, and their tiles more than the tables hold: the sums stop at what those
    // do, so that none overflows and each tile found is one of its group's.
    const uint32_t most = 64u * TABLE * gridDim.x;  // at most 2^30 and a round
    auto add = [&](uint32_t a, uint32_t b) { return min(a + b, most); };
    uint32_t sum = 0;
    for (int e = e0; e < e1; ++e) {
      int beg, n;
      range(e, beg, n);
      sum = add(sum, (uint32_t)tiles_of(n));
    }
    uint32_t upto = sum;
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t v = __shfl_up(upto, d);
      if ((t & 63) >= d) upto = add(upto, v);
    }
    if ((t & 63) == 63) part[t >> 6] = (int)upto;
    upto = __shfl_up(upto, 1);  // of the threads before
    __syncthreads();
    uint32_t total = 0, at = (t & 63) ? upto : 0u;
    for (int w = 0; w < mm16::THREADS / 64; ++w) {
      at = add(at, w < t >> 6 ? (uint32_t)part[w] : 0u);
      total = add(total, (uint32_t)part[w]);
    }
    for (int e = e0; e < e1; ++e) {
      int beg, n;
      range(e, beg, n);
      first[e] = (int)at;
      at = add(at, (uint32_t)tiles_of(n));
    }
    if (t == 0) first[g.groups] = (int)total;
    __syncthreads();
    const int all = __builtin_amdgcn_readfirstlane((int)total);
    count = mm16::worker_tiles(all);
    // The XCDs go through the rounds that all of them take part in from an eighth of the way apart: tiles of large
    // groups, bound by their MFMAs, run beside tiles of small ones, bound by the weights' bytes (8192 rows in 48
    // groups, 7168 x 2048, Zipf: 388 us in one order, 362 so).
    const int whole = all / (int)gridDim.x, from = (int)(blockIdx.x % 8) * whole / 8;
#pragma unroll
    for (int q = 0; q < TABLE; ++q) {
      int x = 64 * q + (t & 63);
      if (MODE != DW && x < whole) x = x + from < whole ? x + from : x + from - whole;
      const int tile = mm16::worker_number() + x * (int)gridDim.x;
      group_nt[q] = mt_of[q] = beg_of[q] = n_of[q] = 0;
      if (tile < all) {
        int lo = 0, hi = g.groups;  // first[lo] <= tile < first[hi]
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (first[mid] <= tile) lo = mid;
          else hi = mid;
        }
        // (rounded up: the last group before the sums stop may have part of its tiles)
        int nt;
        mm16::tile_mn(tile - first[lo], (first[lo + 1] - first[lo] + ntiles - 1) / ntiles, ntiles, mt_of[q], nt);
        group_nt[q] = lo << 16 | nt;
        range(lo, beg_of[q], n_of[q]);
      }
    }
    __syncthreads();  // the slabs' loads overwrite the sums
  }

  __device__ __forceinline__ int entry(const int (&v)[TABLE], int i) const {
    const int q = i >> 6, l = i & 63;
    int r = __builtin_amdgcn_readlane(v[0], l);
#pragma unroll
    for (int x = 1; x < TABLE; ++x) r = q == x ? __builtin_amdgcn_readlane(v[x], l) : r;
    return r;
  }

  // Group, first row and row count of it, and position of this worker's tile i.
  __device__ __forceinline__ void find(int i, int& e, int& beg, int& n, int& mt, int& nt) const {
    const int en = entry(group_nt, i);
    e = en >> 16;
    nt = en & 0xffff;
    mt = entry(mt_of, i);
    beg = entry(beg_of, i);
    n = entry(n_of, i);
  }

  __device__ __forceinline__ mm16::Tile tile(int i) const {
    int e, beg, n, mt, nt;
    find(i, e, beg, n, mt, nt);
    const int m0 = mt * mm16::BM, n0 = nt * mm16::BN;
    mm16::Tile r;
    r.a.ld = g.ld_in;
    r.b.ld = g.ld_other;
    r.cols = mm16::BN;
    if (MODE == DW) {
      r.kc = n;
      r.rows = min(mm16::BM, g.n - m0);
      r.a.base = g.rows_in + (int64_t)beg * g.ld_in + 2 * (int64_t)m0;
      r.a.width = 2u * (uint32_t)(g.n - m0);
      r.b.base = g.other + (int64_t)beg * g.ld_other + 2 * (int64_t)n0;
      r.b.width = 2u * (uint32_t)(g.k - n0);
      r.a.rows = r.b.rows = 0;
    } else {
      r.kc = MODE == FORWARD ? g.k : g.n;
      r.rows = min(mm16::BM, n - m0);
      r.a.base = g.rows_in + (int64_t)(beg + m0) * g.ld_in;
      r.a.rows = r.rows;
      r.a.width = 0;
      const char* w = g.other + (int64_t)e * g.n * g.ld_other;
      if (MODE == FORWARD) {
        r.b.base = w + (int64_t)n0 * g.ld_other;
        r.b.rows = min(mm16::BN, g.n - n0);
        r.b.width = 0;
      } else {
        r.b.base = w + 2 * (int64_t)n0;
        r.b.rows = 0;
        r.b.width = 2u * (uint32_t)(g.k - n0);
      }
      r.once = STREAM && n <= 128;
    }
    return r;
  }

  template <int NB, int WN>
  __device__ __forceinline__ bool epilogue(const mm16::Tile& tl, int i, int wm, int wn,
                                           float16_t (&acc)[NB][WN], int lane) const {
    int e, beg, n, mt, nt;
    find(i, e, beg, n, mt, nt);
    const int m0 = mt * mm16::BM, n0 = nt * mm16::BN;
    const int64_t row0 = MODE == DW ? (int64_t)e * g.n + m0 : beg + m0;
    const int cols = (MODE == FORWARD ? g.n : g.k) - n0;
    if constexpr (KIND == mm16::I8) {
      constexpr int ES = OUT == KQ_DT_F32 ? 4 : 2;
      int8::Finish f{};
      f.sx = g.sx + row0;
      f.sw = g.sw + (int64_t)e * g.n + n0;
      f.out = g.out + row0 * g.ld_out + ES * (int64_t)n0;
      f.ld = g.ld_out;
      f.pieces = true;  // (n and ld_out are multiples of 8 elements)
      int8::finish<NB, WN, OUT, EPI_OFF>(f, tl.rows, min(cols, mm16::BN), wm, wn, acc, lane);
      return tl.rows >= mm16::BM && cols >= mm16::BN;
    }
    char* out = g.out + row0 * g.ld_out + 2 * (int64_t)n0;
    mm16::store16<NB, WN, KIND == mm16::F16>([&](int r) { return out + (uint32_t)r * g.ld_out; }, tl.rows, cols, wm, wn, acc, lane,
                               [](int, int, int, float v) { return v; });
    return tl.rows >= mm16::BM && cols >= mm16::BN;
  }
};

// Rows that belong to no group are zeros (workgroup w of `of` clears its share).
template <int ES = 2>
__device__ __forceinline__ void zero_rows(const Args& g, int cols, int w, int of) {
  const int64_t beg = clamped(g.offsets[0], 0, g.rows), end = clamped(g.offsets[g.groups], beg, g.rows);
  const int64_t before = beg, after = g.rows - end;
  for (int64_t i = w; i < before + after; i += of) {
    char* p = g.out + (i < before ? i : end + i - before) * g.ld_out;
    for (int c = (int)threadIdx.x * (16 / ES); c < cols; c += (int)blockDim.x * (16 / ES))
      *reinterpret_cast<mm16::u32x4_t*>(p + ES * (int64_t)c) = mm16::u32x4_t{0u, 0u, 0u, 0u};
  }
}

template <int MODE, int KIND, bool STREAM, int OUT = 0>
__global__ __launch_bounds__(mm16::THREADS, 1) void grouped_kernel(Args g) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[mm16::LDS_BYTES];
  using Mine = Problem<MODE, KIND, STREAM, OUT>;
  Mine p;
  p.g = g;
  p.setup(lds);
  if (MODE != DW) zero_rows<KIND == mm16::I8 && OUT == KQ_DT_F32 ? 4 : 2>(g, MODE == FORWARD ? g.n : g.k, (int)blockIdx.x, (int)gridDim.x);
  mm16::Core<MODE == DW, MODE != FORWARD, KIND, MODE == DW ? mm16::WHOLE : mm16::SMALL_ROWS, true, STREAM, Mine> core(p, lds);
  core.run();
}

// Workgroups of a call, and whether its weights stream.
template <int MODE>
static hipError_t plan(const Args& g, hipStream_t st, int64_t& grid, bool& stream) {
  int dev = 0, cus = 0;
  hipError_t e = st ? hipStreamGetDevice(st, &dev) : hipGetDevice(&dev);
  if (e == hipSuccess) e = hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev);
  if (e != hipSuccess) return e;
  grid = cus >= 8 ? cus / 8 * 8 : 8;
  // a worker's table holds 256 tiles: more workers where there may be more
  const int64_t row_tiles = MODE == DW ? (int64_t)g.groups * ((g.n + mm16::BM - 1) / mm16::BM)
                                       : g.rows / mm16::BM + (g.rows < g.groups ? g.rows : g.groups);
  const int64_t most = row_tiles * (((MODE == FORWARD ? g.n : g.k) + mm16::BN - 1) / mm16::BN);
  grid *= most > 0 ? (most + grid * 64 * TABLE - 1) / (grid * 64 * TABLE) : 1;
  stream = (int64_t)g.groups * g.n * g.k * 2 > LAST_LEVEL_CACHE;
  return hipSuccess;
}

}  // namespace grouped
}  // namespace kq

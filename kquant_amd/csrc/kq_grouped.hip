// Matrix products grouped by expert with ragged sizes: rows sorted by group
// times that group's dense 16-bit weight, and both gradients.
//
//   forward  y[r]  = W_g x[r]                 for the rows r of group g
//   dx       dx[r] = W_g^T dy[r]
//   dw       dW_g  = sum over r of dy[r] x[r]^T
//
// All three run on the tiles of kq_mm16.h: the weight is read along its rows in
// the forward pass and across them for dx, and dw contracts over the rows of a
// group, both operands read across.  Group sizes stay on the device (offsets),
// so each workgroup numbers the tiles itself.
#include "kq_internal.h"
#include "kq_mm16.h"

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
};

constexpr int64_t LAST_LEVEL_CACHE = 256ll << 20;
constexpr int TABLE = 4;  // 64 tiles of a worker each

__shared__ __attribute__((aligned(16))) unsigned char lds[mm16::LDS_BYTES];

// Offsets are device data: clamped to the rows there are, so that no value of
// them reads or writes outside.
__device__ __forceinline__ int64_t clamped(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : v > hi ? hi : v; }

// STREAM: the weights are more than the last-level cache holds.
template <int MODE, bool F16, bool STREAM>
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
  __device__ __forceinline__ void setup() {
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
    char* out = g.out + row0 * g.ld_out + 2 * (int64_t)n0;
    mm16::store16<NB, WN, F16>([&](int r) { return out + (uint32_t)r * g.ld_out; }, tl.rows, cols, wm, wn, acc, lane,
                               [](int, int, int, float v) { return v; });
    return tl.rows >= mm16::BM && cols >= mm16::BN;
  }
};

// Rows that belong to no group are zeros.
__device__ __forceinline__ void zero_rows(const Args& g, int cols) {
  const int64_t beg = clamped(g.offsets[0], 0, g.rows), end = clamped(g.offsets[g.groups], beg, g.rows);
  const int64_t before = beg, after = g.rows - end;
  for (int64_t i = blockIdx.x; i < before + after; i += gridDim.x) {
    char* p = g.out + (i < before ? i : end + i - before) * g.ld_out;
    for (int c = (int)threadIdx.x * 8; c < cols; c += mm16::THREADS * 8)
      *reinterpret_cast<mm16::u32x4_t*>(p + 2 * (int64_t)c) = mm16::u32x4_t{0u, 0u, 0u, 0u};
  }
}

template <int MODE, bool F16, bool STREAM>
__global__ __launch_bounds__(mm16::THREADS, 1) void grouped_kernel(Args g) {
  Problem<MODE, F16, STREAM> p;
  p.g = g;
  p.setup();
  if (MODE != DW) zero_rows(g, MODE == FORWARD ? g.n : g.k);
  mm16::Core<MODE == DW, MODE != FORWARD, F16, MODE == DW ? mm16::WHOLE : mm16::SMALL_ROWS, true,
             STREAM, Problem<MODE, F16, STREAM>> core(p, lds);
  core.run();
}

template <int MODE>
static hipError_t launch(int dtype, const Args& g, hipStream_t st) {
  int dev = 0, cus = 0;
  hipError_t e = st ? hipStreamGetDevice(st, &dev) : hipGetDevice(&dev);
  if (e == hipSuccess) e = hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev);
  if (e != hipSuccess) return e;
  int64_t grid = cus >= 8 ? cus / 8 * 8 : 8;
  // a worker's table holds 256 tiles: more workers where there may be more
  const int64_t row_tiles = MODE == DW ? (int64_t)g.groups * ((g.n + mm16::BM - 1) / mm16::BM)
                                       : g.rows / mm16::BM + (g.rows < g.groups ? g.rows : g.groups);
  const int64_t most = row_tiles * (((MODE == FORWARD ? g.n : g.k) + mm16::BN - 1) / mm16::BN);
  grid *= most > 0 ? (most + grid * 64 * TABLE - 1) / (grid * 64 * TABLE) : 1;
  const bool stream = (int64_t)g.groups * g.n * g.k * 2 > LAST_LEVEL_CACHE;
  auto run = [&](auto streamed) {
    constexpr bool S = MODE != DW && streamed.value;
    if (dtype == KQ_DT_F16) grouped_kernel<MODE, true, S><<<(unsigned)grid, mm16::THREADS, 0, st>>>(g);
    else grouped_kernel<MODE, false, S><<<(unsigned)grid, mm16::THREADS, 0, st>>>(g);
  };
  if (stream) run(std::true_type{});
  else run(std::false_type{});
  return hipGetLastError();
}

static int check(const char* fn, int dtype, int64_t rows, int groups, int64_t n, int64_t k, int64_t ld_n, int64_t ld_k,
                 const int64_t* offsets, const void* a, const void* b, const void* c) {
  if (dtype != KQ_DT_BF16 && dtype != KQ_DT_F16) return kq_fail(KQ_ERR_INVALID, "%s: dtype must be bf16 or f16", fn);
  if (rows < 0 || groups < 1 || n <= 0 || k <= 0 || n % 8 || k % 8 || ld_n < n || ld_k < k || ld_n % 8 || ld_k % 8)
    return kq_fail(KQ_ERR_INVALID,
                   "%s: need groups >= 1, n %% 8 == 0, k %% 8 == 0, row strides of at least n and k, multiples of 8 "
                   "(rows=%lld groups=%d n=%lld k=%lld strides %lld, %lld)",
                   fn, (long long)rows, groups, (long long)n, (long long)k, (long long)ld_n, (long long)ld_k);
  const int64_t tiles_n = (n + 255) / 256, tiles_k = (k + 255) / 256;
  if (groups > MAX_GROUPS || rows > INT32_MAX / 2 || ld_n > mm16::MAX_LD || ld_k > mm16::MAX_LD ||
      (int64_t)groups * tiles_n * tiles_k > INT32_MAX / 2 ||
      (rows / 256 + groups) * (tiles_n > tiles_k ? tiles_n : tiles_k) > INT32_MAX / 2)
    return kq_fail(KQ_ERR_LIMIT, "%s: at most %d groups, 2^30 rows and tiles, rows of 2^22 elements", fn, MAX_GROUPS);
  if (!offsets || kq_misaligned(offsets, 8)) return kq_fail(KQ_ERR_INVALID, "%s: offsets must be int64 on the device", fn);
  if (kq_misaligned(a, 16) || kq_misaligned(b, 16) || kq_misaligned(c, 16))
    return kq_fail(KQ_ERR_INVALID, "%s: operands must be 16-byte aligned", fn);
  return KQ_OK;
}

}  // namespace grouped
}  // namespace kq

using namespace kq;

extern "C" int kq_grouped_linear(int dtype, const void* x, int64_t ldx, int64_t rows, const int64_t* offsets, int groups,
                                 const void* w, int64_t n, int64_t k, void* y, int64_t ldy, void* stream) {
  if (int rc = grouped::check("kq_grouped_linear", dtype, rows, groups, n, k, ldy, ldx, offsets, x, w, y)) return rc;
  if (rows == 0) return KQ_OK;
  const grouped::Args g{(const char*)x, (const char*)w, (char*)y, (uint32_t)(2 * ldx), (uint32_t)(2 * k),
                        (uint32_t)(2 * ldy), offsets, rows, groups, (int)n, (int)k};
  return kq_check_launch(grouped::launch<grouped::FORWARD>(dtype, g, (hipStream_t)stream), "kq_grouped_linear");
}

extern "C" int kq_grouped_linear_dx(int dtype, const void* dy, int64_t lddy, int64_t rows, const int64_t* offsets,
                                    int groups, const void* w, int64_t n, int64_t k, void* dx, int64_t lddx,
                                    void* stream) {
  if (int rc = grouped::check("kq_grouped_linear_dx", dtype, rows, groups, n, k, lddy, lddx, offsets, dy, w, dx)) return rc;
  if (rows == 0) return KQ_OK;
  const grouped::Args g{(const char*)dy, (const char*)w, (char*)dx, (uint32_t)(2 * lddy), (uint32_t)(2 * k),
                        (uint32_t)(2 * lddx), offsets, rows, groups, (int)n, (int)k};
  return kq_check_launch(grouped::launch<grouped::DX>(dtype, g, (hipStream_t)stream), "kq_grouped_linear_dx");
}

extern "C" int kq_grouped_linear_dw(int dtype, const void* dy, int64_t lddy, const void* x, int64_t ldx, int64_t rows,
                                    const int64_t* offsets, int groups, int64_t n, int64_t k, void* dw, void* stream) {
  if (int rc = grouped::check("kq_grouped_linear_dw", dtype, rows, groups, n, k, lddy, ldx, offsets, dy, x, dw)) return rc;
  const grouped::Args g{(const char*)dy, (const char*)x, (char*)dw, (uint32_t)(2 * lddy), (uint32_t)(2 * ldx),
                        (uint32_t)(2 * k), offsets, rows, groups, (int)n, (int)k};
  return kq_check_launch(grouped::launch<grouped::DW>(dtype, g, (hipStream_t)stream), "kq_grouped_linear_dw");
}
